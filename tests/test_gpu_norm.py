"""GPU tier: the block norms, forward and backward, against the 64-bit oracle and against differences.

Bounds: with u = 2^-24, a thread adds at most 64 products of a row and the tree over threads has at most 10 levels, so a sum of
H magnitudes is off by at most 80 u of itself; rstd by half of that, its cube by 120 u; products and differences add a few
each.  Every value is then within 512 u of its `size` (the formula with all terms' magnitudes added), plus half a step of its
type.  Sums over tokens add at most T/148 + T/1184 + 10 terms in a row, which stays below that for the sizes here."""
import pytest
import torch

from oracle import dense_oracle as orc
from pyhip_b200 import fused_post_norm, fused_pre_norm, quantize_int8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
C = 512 * 2.0 ** -24
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -140}


def _near(x, ref, size, what):
    bound = torch.finfo(x.dtype).eps / 2 * ref.abs() + C * size + TINY[x.dtype]
    off = (x.double() - ref).abs() - bound
    assert x.shape == ref.shape and torch.isfinite(x).all() and float(off.detach().max()) <= 0, \
        f"{what}: {int((off > 0).sum())} of {off.numel()} out of bounds, worst {float(off.detach().max()):.3e}"


def _randn(*shape, seed, dtype, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(DEV)


def _inputs(T, H, dtype, pdtype, post, gate, nxt, residual=True, seed=0):
    lead = T if isinstance(T, tuple) else (T,)
    i = dict(y=_randn(*lead, H, seed=seed, dtype=dtype), residual=_randn(*lead, H, seed=seed + 1, dtype=dtype, scale=2.0) if residual else None,
             weight=_randn(H, seed=seed + 2, dtype=pdtype, scale=0.2, shift=1.0) if post else None, gate=None,
             next_weight=_randn(H, seed=seed + 3, dtype=pdtype, scale=0.2, shift=1.0) if nxt else None)
    if gate:
        i["gate"] = _randn(*dict(channel=(H,), token=(*lead, 1), full=(*lead, H))[gate], seed=seed + 4, dtype=pdtype, scale=0.5, shift=0.3)
    return i


WIDTHS = [(1, 1), (3, 7), (2, 32), (70, 64), (33, 288), (5, 1001), (40, 2880), (3, 4104), (9, 7168), (2, 8193), (2, 16384), (1, 16383),
          (700, 2880), (593, 520), (600, 1000), (1300, 7168), (595, 16384)]        # the last ones take the ring where it applies


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H", WIDTHS)
def test_forward_matches_64_bits(T, H, dtype):
    for k, (post, gate, nxt, pdtype) in enumerate([(True, "channel", True, torch.float32), (True, None, False, dtype), (False, "token", True, dtype),
                                                   (True, "full", True, dtype), (False, "full", False, torch.float32)]):
        i = _inputs(T, H, dtype, pdtype, post, gate, nxt, seed=T + H + k)
        o = orc.block_norm(i["y"], i["residual"], i["weight"], i["gate"], 0.75, 1e-5, i["next_weight"])
        r = fused_post_norm(i["y"], i["residual"], i["weight"], gate=i["gate"], residual_scale=0.75, eps=1e-5, next_weight=i["next_weight"])
        h, n = r if nxt else (r, None)
        _near(h, o["h"], o["h_size"], "h")
        if nxt:
            _near(n, o["n"], o["n_size"], "n")
    i = _inputs(T, H, dtype, dtype, False, None, True, seed=T)
    o = orc.block_norm(i["y"], None, None, None, 1.0, 1e-6, i["next_weight"])
    _near(fused_pre_norm(i["y"], i["next_weight"]), o["n"], o["n_size"], "pre n")
    o = orc.block_norm(i["y"], i["residual"], None, None, 1.0, 1e-6, i["next_weight"])
    n, h = fused_pre_norm(i["y"], i["next_weight"], residual=i["residual"])
    _near(n, o["n"], o["n_size"], "pre n")
    _near(h, o["h"], o["h_size"], "pre h")


def _grads(i, r, dh, dn):
    outs, seeds = [], []
    for o, g in zip(r if isinstance(r, tuple) else (r,), (dh, dn)):
        if g is not None:
            outs.append(o), seeds.append(g)
    names = [k for k in i if i[k] is not None]
    return dict(zip(names, torch.autograd.grad(outs, [i[k] for k in names], seeds, allow_unused=True)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H", [(1, 1), (3, 7), (70, 64), (300, 288), (5, 1001), (700, 2880), (3, 4104), (160, 7168), (2, 8193), (2, 16384), (1, 16383),
                                 (593, 520), (1300, 1000), (600, 4104), (605, 7168), (620, 8192), (595, 16384)])
def test_backward_matches_64_bits(T, H, dtype):
    for k, (post, gate, nxt, pdtype) in enumerate([(True, "channel", True, torch.float32), (True, None, False, dtype), (False, "token", True, dtype),
                                                   (True, "token", True, dtype), (True, "full", True, dtype), (False, "full", False, torch.float32),
                                                   (False, "channel", True, dtype)]):
        i = _inputs(T, H, dtype, pdtype, post, gate, nxt, seed=T + H + k)
        o = orc.block_norm(i["y"], i["residual"], i["weight"], i["gate"], 0.75, 1e-5, i["next_weight"])
        for t in i.values():
            if t is not None:
                t.requires_grad_(True)
        dh, dn = _randn(T, H, seed=k, dtype=dtype), _randn(T, H, seed=k + 50, dtype=dtype) if nxt else None
        r = fused_post_norm(i["y"], i["residual"], i["weight"], gate=i["gate"], residual_scale=0.75, eps=1e-5, next_weight=i["next_weight"])
        got = _grads(i, r, dh, dn)
        want = orc.block_norm_grads(o, i["residual"], i["weight"], i["gate"], 0.75, i["next_weight"], dh, dn)
        assert got.keys() == want.keys()
        for name in want:
            assert got[name].dtype == i[name].dtype
            _near(got[name], *want[name], f"{name} (case {k})")


@pytest.mark.parametrize("T,H", [(5, 96), (300, 2880), (40, 7168), (3, 16384)])
@pytest.mark.parametrize("gate", ["channel", "token", "full"])
def test_parameters_of_different_types(T, H, gate):
    """Weights, next weights and gates each fp32 or of the rows' type."""
    bf, f = torch.bfloat16, torch.float32
    for k, (wt, gt, nt) in enumerate([(f, bf, bf), (bf, bf, f), (bf, f, bf), (f, f, bf), (f, bf, f)]):
        i = _inputs(T, H, bf, f, True, gate, True, seed=T + k)
        i = dict(i, weight=i["weight"].to(wt), gate=i["gate"].to(gt), next_weight=i["next_weight"].to(nt))
        o = orc.block_norm(i["y"], i["residual"], i["weight"], i["gate"], 0.75, 1e-5, i["next_weight"])
        for t in i.values():
            t.requires_grad_(True)
        dh, dn = _randn(T, H, seed=k, dtype=bf), _randn(T, H, seed=k + 50, dtype=bf)
        r = fused_post_norm(i["y"], i["residual"], i["weight"], gate=i["gate"], residual_scale=0.75, eps=1e-5, next_weight=i["next_weight"])
        _near(r[0].detach(), o["h"], o["h_size"], "h")
        _near(r[1].detach(), o["n"], o["n_size"], "n")
        got = _grads(i, r, dh, dn)
        want = orc.block_norm_grads(o, i["residual"], i["weight"], i["gate"], 0.75, i["next_weight"], dh, dn)
        for name in want:
            assert got[name].dtype == i[name].dtype
            _near(got[name], want[name][0].detach(), want[name][1].detach(), f"{name} (case {k})")


def test_formula_matches_differences():
    """The oracle's gradients (64 bits) against central differences of its forward."""
    i = {k: None if v is None else v.double().cpu() for k, v in _inputs(3, 5, torch.float32, torch.float32, True, "token", True).items()}
    dh, dn = torch.randn(3, 5, dtype=torch.float64), torch.randn(3, 5, dtype=torch.float64)

    def loss(j):
        o = orc.block_norm(j["y"], j["residual"], j["weight"], j["gate"], 0.5, 1e-5, j["next_weight"])
        return float((o["h"] * dh).sum() + (o["n"] * dn).sum())

    want = orc.block_norm_grads(orc.block_norm(i["y"], i["residual"], i["weight"], i["gate"], 0.5, 1e-5, i["next_weight"]), i["residual"],
                                i["weight"], i["gate"], 0.5, i["next_weight"], dh, dn)
    for name, (g, _) in want.items():
        for at in range(i[name].numel()):
            d = []
            for step in (1e-5, -1e-5):
                j = dict(i, **{name: i[name].clone()})
                j[name].view(-1)[at] += step
                d.append(loss(j))
            # central differences: the third derivatives here are below 100, so 1e-10 * 100 / 6, and 1e-15 * |loss| / 1e-5
            assert abs((d[0] - d[1]) / 2e-5 - float(g.reshape(-1)[at])) < 1e-7


def test_partial_gradients_and_expanded_ones():
    """Only some gradients wanted, one of two outputs used, and an upstream gradient that is an expanded scalar."""
    i = _inputs(20, 96, torch.float32, torch.float32, True, "channel", True, seed=3)
    o = orc.block_norm(i["y"], i["residual"], i["weight"], i["gate"], 1.0, 1e-6, i["next_weight"])
    ones = torch.ones(20, 96, device=DEV)
    for name in i:
        j = {k: v.detach().clone().requires_grad_(k == name) for k, v in i.items()}
        h, n = fused_post_norm(j["y"], j["residual"], j["weight"], gate=j["gate"], next_weight=j["next_weight"])
        (h.sum() + n.sum()).backward()
        _near(j[name].grad, *orc.block_norm_grads(o, i["residual"], i["weight"], i["gate"], 1.0, i["next_weight"], ones, ones)[name], name)
    j = {k: v.detach().clone().requires_grad_(True) for k, v in i.items()}
    h, n = fused_post_norm(j["y"], j["residual"], j["weight"], gate=j["gate"], next_weight=j["next_weight"])
    n.sum().backward()
    want = orc.block_norm_grads(o, i["residual"], i["weight"], i["gate"], 1.0, i["next_weight"], None, ones)
    for name in want:
        _near(j[name].grad, *want[name], name)
    j = {k: v.detach().clone().requires_grad_(True) for k, v in i.items()}
    h, n = fused_post_norm(j["y"], j["residual"], j["weight"], gate=j["gate"], next_weight=j["next_weight"])
    h.sum().backward()
    want = orc.block_norm_grads(o, i["residual"], i["weight"], i["gate"], 1.0, i["next_weight"], ones, None)
    for name in want:
        _near(j[name].grad, *want[name], name)
    x = i["y"].detach().clone().requires_grad_(True)
    w = i["next_weight"].detach().clone().requires_grad_(True)
    fused_pre_norm(x, w).sum().backward()
    o = orc.block_norm(x.detach(), None, None, None, 1.0, 1e-6, w.detach())
    want = orc.block_norm_grads(o, None, None, None, 1.0, w.detach(), None, ones)
    _near(x.grad, *want["y"], "x")
    _near(w.grad, *want["next_weight"], "w")


def test_a_tensor_used_twice_gets_both_gradients():
    x = _randn(12, 64, seed=1, dtype=torch.float32).requires_grad_(True)
    w = _randn(64, seed=2, dtype=torch.float32, shift=1.0).requires_grad_(True)
    h, n = fused_post_norm(x, x, w, gate=x, next_weight=w)
    one = torch.ones_like(h)
    gx, gw = torch.autograd.grad([h, n], [x, w], [one, one])
    xd, wd = x.detach(), w.detach()
    o = orc.block_norm(xd, xd, wd, xd, 1.0, 1e-6, wd)
    want = orc.block_norm_grads(o, xd, wd, xd, 1.0, wd, one, one)
    parts = [want[k] for k in ("y", "residual", "gate")]
    _near(gx, sum(p[0] for p in parts), sum(p[1] + p[0].abs() for p in parts), "x")
    parts = [want[k] for k in ("weight", "next_weight")]
    _near(gw, sum(p[0] for p in parts), sum(p[1] + p[0].abs() for p in parts), "w")


@pytest.mark.parametrize("H", [64, 100, 2880])
def test_strides_shapes_and_empty(H):
    big = _randn(30, H + 24, seed=1, dtype=torch.bfloat16)
    res = _randn(30, 2 * H, seed=2, dtype=torch.bfloat16)
    gate = _randn(30, H + 8, seed=3, dtype=torch.bfloat16)
    w = _randn(H, seed=4, dtype=torch.bfloat16, shift=1.0)
    for a, b, g in ((big[:, 8:H + 8], res[:, :H], gate[:, 8:]), (big[:, 3:H + 3], res[:, H:], gate[:, 1:H + 1]), (big[::3, :H], res[::3, :H], gate[::3, :H]),
                    (big[:1, :H].expand(30, H), res[:, :H], gate[:1, :H].expand(30, H))):
        want = fused_post_norm(a.contiguous(), b.contiguous(), w, gate=g.contiguous(), next_weight=w)
        got = fused_post_norm(a, b, w, gate=g, next_weight=w)
        # the wide and the narrow accesses add a row's squares in another order: not the same bits, the same bounds
        o = orc.block_norm(a, b, w, g, 1.0, 1e-6, w)
        for r in (want, got):
            _near(r[0], o["h"], o["h_size"], "h")
            _near(r[1], o["n"], o["n_size"], "n")
    a, b = big[:, 3:H + 3].detach().requires_grad_(True), res[:, H:].detach().requires_grad_(True)
    ga, gb = torch.autograd.grad(fused_post_norm(a, b, w), [a, b], torch.ones(30, H, device=DEV, dtype=torch.bfloat16))
    o = orc.block_norm(a.detach(), b.detach(), w, None, 1.0, 1e-6)
    want = orc.block_norm_grads(o, b, w, None, 1.0, None, torch.ones(30, H, device=DEV))
    _near(ga, *want["y"], "y")
    _near(gb, *want["residual"], "residual")
    x3 = _randn(2, 5, H, seed=6, dtype=torch.bfloat16)
    assert torch.equal(fused_pre_norm(x3, w), fused_pre_norm(x3.view(10, H), w).view(2, 5, H))
    tok = _randn(2, 5, 1, seed=7, dtype=torch.bfloat16)
    assert torch.equal(fused_post_norm(x3, x3, w, gate=tok), fused_post_norm(x3.view(10, H), x3.view(10, H), w, gate=tok.view(10, 1)).view(2, 5, H))
    h, n = fused_post_norm(x3[:0], x3[:0], w, next_weight=w)
    assert h.shape == n.shape == (0, 5, H)
    e, we = x3[:0].detach().requires_grad_(True), w.detach().clone().requires_grad_(True)
    gs = torch.autograd.grad(fused_post_norm(e, e.detach(), we, next_weight=we), [e, we], [torch.zeros_like(h)] * 2)
    assert gs[0].shape == (0, 5, H) and (gs[1] == 0).all()
    for g in (tok[:0], x3[:0], w):
        assert fused_post_norm(x3[:0], x3[:0], w, gate=g).shape == (0, 5, H)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H", [(1, 16), (5, 1001), (40, 2880), (3, 16384)])
def test_int8_rows(T, H, dtype):
    """The scale of a row is the largest |n| / 127 of a row within C of the exact one; a value is within half a step of it."""
    i = _inputs(T, H, dtype, dtype, True, "channel", True, seed=T)
    o = orc.block_norm(i["y"], i["residual"], i["weight"], i["gate"], 1.0, 1e-6, i["next_weight"])
    h, q, s = fused_post_norm(i["y"], i["residual"], i["weight"], gate=i["gate"], next_weight=i["next_weight"], quant="int8")
    _near(h, o["h"], o["h_size"], "h")
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and s.shape == (T,)
    amax, slack = o["n"].abs().amax(-1), C * o["n_size"].amax(-1)
    assert ((s.double() * 127 - amax).abs() <= slack + amax * 2.0 ** -23).all()
    back = q.double() * s.double()[:, None]
    assert ((back - o["n"]).abs() <= s.double()[:, None] * 0.5 + C * o["n_size"]).all()
    assert q.abs().amax(-1).eq(127).all()
    # without a norm in between the rows are those of the quantiser
    x = i["y"]
    one = torch.ones(H, device=DEV)
    q2, s2 = fused_pre_norm(x, one, quant="int8")
    q3, s3, h3 = fused_pre_norm(x, one, residual=torch.zeros_like(x), quant="int8")
    # a row whose copies with the residual do not fit the ring adds its squares in another order: both sides' largest value is
    # within C of the exact one (and a rounding more in the division), so the scales within twice that of one another, and a
    # quotient of at most 127 moves by less than 127 * 2 * C < 0.01, one step of the grid at most
    assert ((s2 - s3).abs() <= 2 * (C + 2.0 ** -23) * s2).all() and (q2.int() - q3.int()).abs().max() <= 1 and torch.equal(h3, x)
    qq, ss = quantize_int8(x)
    assert (q2.int() - qq.int()).abs().max() <= 1


def test_special_values_stay_in_their_row():
    i = _inputs(9, 96, torch.bfloat16, torch.bfloat16, True, "token", True, seed=8)
    clean = fused_post_norm(i["y"], i["residual"], i["weight"], gate=i["gate"], next_weight=i["next_weight"])
    y = i["y"].clone()
    y[3, 4], y[5, 6] = float("nan"), float("inf")
    y[7] = 0
    got = fused_post_norm(y, i["residual"], i["weight"], gate=i["gate"], next_weight=i["next_weight"])
    rows = [0, 1, 2, 4, 6, 8]
    for a, b in zip(got, clean):
        assert torch.equal(a[rows], b[rows])
    assert got[1][3].isnan().all() and got[1][5].isnan().any()
    assert torch.isfinite(got[0][7]).all() and torch.isfinite(got[1][7]).all()          # a row of zeros: rstd = 1 / sqrt(eps)
    z = torch.zeros(3, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(64, device=DEV)
    assert (fused_pre_norm(z, w) == 0).all()
    q, s = fused_pre_norm(z, w, quant="int8")
    assert (q == 0).all() and (s == 2.0 ** -100).all()


def test_same_bits_every_time_and_in_graphs():
    i = _inputs(500, 2880, torch.bfloat16, torch.float32, True, "channel", True, seed=4)
    for t in i.values():
        t.requires_grad_(True)
    dh, dn = _randn(500, 2880, seed=1, dtype=torch.bfloat16), _randn(500, 2880, seed=2, dtype=torch.bfloat16)

    def step():
        r = fused_post_norm(i["y"], i["residual"], i["weight"], gate=i["gate"], next_weight=i["next_weight"])
        return [*r, *torch.autograd.grad(r, list(i.values()), [dh, dn])]

    first = [t.detach().clone() for t in step()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(), first))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, first))


def test_refusals():
    x, w = _randn(4, 64, seed=1, dtype=torch.bfloat16), _randn(64, seed=2, dtype=torch.bfloat16)
    for call in (lambda: fused_pre_norm(x, w[:32]), lambda: fused_pre_norm(x, w.half()), lambda: fused_pre_norm(x, None),
                 lambda: fused_pre_norm(x, w, residual=x[:2]), lambda: fused_pre_norm(x, w, residual=x.float()),
                 lambda: fused_pre_norm(x, w, quant="fp8"), lambda: fused_post_norm(x, None, w), lambda: fused_post_norm(x, x, w, gate=w[:4]),
                 lambda: fused_post_norm(x, x, w, quant="int8"), lambda: fused_post_norm(x, x.cpu(), w),
                 lambda: fused_pre_norm(torch.empty(1, 16385, device=DEV), torch.empty(16385, device=DEV))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: fused_pre_norm(x.double(), w.double()), lambda: fused_post_norm(x, x, w, gate=w.half())):
        with pytest.raises(TypeError):
            call()
    w.requires_grad_(True)
    with pytest.raises(RuntimeError):
        fused_pre_norm(x, w, quant="int8")
    with torch.no_grad():
        fused_pre_norm(x, w, quant="int8")
