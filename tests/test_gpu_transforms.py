"""GPU tier: the dense operators under what torch lays over a call -- forward-mode derivatives, tracing, wrapped tensors, lazy
negation.  Where an operator cannot take part it has to say so: a result without its tangent or a trace without the kernel is a
wrong answer."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from pyhip_b200 import fused_post_norm, fused_pre_norm, fused_router, linear_int8, quantize_int8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _tensors():
    g = torch.Generator().manual_seed(3)
    t = dict(x=torch.randn(6, 64, generator=g), r=torch.randn(6, 64, generator=g), w=torch.randn(64, generator=g) + 2, g=torch.randn(6, 1, generator=g),
             n=torch.randn(64, generator=g) + 2, logits=torch.randn(6, 16, generator=g), ws=torch.rand(32, generator=g) + 0.1, b=torch.randn(32, generator=g))
    t = {k: v.to(DEV) for k, v in t.items()}
    t["q"], t["qs"] = quantize_int8(t["x"])
    t["iw"] = torch.randint(-127, 128, (32, 64), generator=g, dtype=torch.int8).to(DEV)
    t["mask"] = torch.tensor([True, True, False, True, True, True], device=DEV)
    t["cu"] = torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV)
    return t


# every call with the names of the float tensors that it takes
CALLS = {
    "pre_norm": (lambda t: fused_pre_norm(t["x"], t["w"], residual=t["r"]), "x w r"),
    "pre_norm_int8": (lambda t: fused_pre_norm(t["x"], t["w"], residual=t["r"], quant="int8"), "x w r"),
    "post_norm": (lambda t: fused_post_norm(t["x"], t["r"], t["w"], gate=t["g"], next_weight=t["n"]), "x r w g n"),
    "router": (lambda t: fused_router(t["logits"], 3, token_mask=t["mask"], cu_seqlens=t["cu"]), "logits"),
    "quantize": (lambda t: quantize_int8(t["x"]), "x"),
    "linear": (lambda t: linear_int8(t["x"], t["iw"], t["ws"], bias=t["b"]), "x ws b"),
    "linear_int8_rows": (lambda t: linear_int8(t["q"], t["iw"], t["ws"], x_scale=t["qs"]), "ws qs"),
}


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    call, names = CALLS[name]
    t = _tensors()
    for key in names.split():
        with fw.dual_level():
            d = dict(t, **{key: fw.make_dual(t[key], torch.ones_like(t[key]))})
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(d)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):      # forward mode goes on there
                call(d)
        call(t)


def test_forward_mode_over_the_backward_pass_is_refused():
    t = _tensors()
    for call, leaf in ((lambda x: fused_pre_norm(x, t["w"]), t["x"]), (lambda x: fused_router(x, 3).topk_weights, t["logits"])):
        x = leaf.clone().requires_grad_(True)
        out = call(x)
        with fw.dual_level():
            up = fw.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, up)


@pytest.mark.parametrize("name", CALLS)
def test_tracing_is_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    call, names = CALLS[name]
    t = _tensors()
    key = names.split()[0]

    def f(v):
        return tuple(call(dict(t, **{key: v}))) if name != "linear" and name != "linear_int8_rows" else call(dict(t, **{key: v}))

    with torch.no_grad():
        for trace in (lambda: torch.jit.trace(f, (t[key],), check_trace=False), lambda: make_fx(f)(t[key]), lambda: make_fx(f, pre_dispatch=True)(t[key])):
            with pytest.raises(RuntimeError, match="trac"):
                trace()


def test_tracing_the_backward_pass_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    t = _tensors()
    for call, leaf in ((lambda x: fused_pre_norm(x, t["w"]), t["x"]), (lambda x: fused_router(x, 3).topk_weights, t["logits"])):
        x = leaf.clone().requires_grad_(True)
        out = call(x)
        with pytest.raises(RuntimeError, match="trac"):
            make_fx(lambda up: torch.autograd.grad(out, x, up))(torch.ones_like(out))


class Wrapped(torch.Tensor):
    """A tensor that holds another one and has no memory of its own."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    def __init__(self, t):
        self.inner = t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        return func(*(a.inner if isinstance(a, cls) else a for a in args), **(kwargs or {}))


@pytest.mark.parametrize("name", CALLS)
def test_wrapped_tensors_are_refused(name):
    call, names = CALLS[name]
    t = _tensors()
    extra = dict(router=" mask cu", linear=" iw", linear_int8_rows=" q iw").get(name, "")
    for key in (names + extra).split():
        with torch.no_grad(), pytest.raises((TypeError, RuntimeError)):
            call(dict(t, **{key: Wrapped(t[key])}))
    with torch.no_grad(), pytest.raises((TypeError, RuntimeError)):
        torch.func.vmap(lambda v: call(dict(t, **{names.split()[-1]: v})))(torch.stack([t[names.split()[-1]]] * 2))


def test_batched_gradients_are_refused():
    t = _tensors()
    x = t["x"].clone().requires_grad_(True)
    out = fused_pre_norm(x, t["w"])
    with pytest.raises((TypeError, RuntimeError)):
        torch.autograd.grad(out, x, torch.ones(3, *out.shape, device=DEV), is_grads_batched=True)


def test_upstream_gradients_that_are_known_to_be_zero():
    t = _tensors()
    x, w = t["x"].clone().requires_grad_(True), t["w"].clone().requires_grad_(True)
    n, h = fused_pre_norm(x, w, residual=t["r"])
    zero = torch._efficientzerotensor(n.shape, dtype=n.dtype, device=n.device)
    got = torch.autograd.grad([n, h], [x, w], [zero, torch.ones_like(h)], retain_graph=True)
    want = torch.autograd.grad([n, h], [x, w], [torch.zeros_like(n), torch.ones_like(h)])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_sparse_tensors_are_refused():
    t = _tensors()
    for key in ("x", "w"):
        with pytest.raises((TypeError, RuntimeError)):
            fused_pre_norm(**{"x": t["x"], "weight": t["w"], {"x": "x", "w": "weight"}[key]: t[key].to_sparse()})


@pytest.mark.parametrize("name", CALLS)
def test_lazily_negated_tensors_are_read_as_such(name):
    """The imaginary part of a conjugate is a view with a negation that is still to be made."""
    call, names = CALLS[name]
    t = _tensors()
    for key in names.split():
        for v in (torch.complex(torch.zeros_like(t[key]), -t[key]).conj().imag, torch._neg_view(-t[key])):      # strided and dense
            assert v.is_neg() and torch.equal(v, t[key])
            with torch.no_grad():
                got, want = call(dict(t, **{key: v})), call(t)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert torch.equal(a, b)


def test_lazily_negated_gradients_are_read_as_such():
    t = _tensors()
    for call, leaf in ((lambda x: fused_pre_norm(x, t["w"]), t["x"]), (lambda x: fused_router(x, 3).topk_weights, t["logits"]),
                       (lambda x: fused_router(x, 3).z_loss, t["logits"])):
        x = leaf.clone().requires_grad_(True)
        up = torch.randn_like(call(x))
        want, = torch.autograd.grad(call(x), x, up)
        for v in (torch.complex(torch.zeros_like(up), -up).conj().imag, torch._neg_view(-up)):
            assert v.is_neg()
            assert torch.equal(torch.autograd.grad(call(x), x, v)[0], want)


def test_a_learned_residual_scale_is_refused():
    """residual_scale is a number: a parameter in its place would train without a gradient."""
    t = _tensors()
    p = torch.nn.Parameter(torch.tensor(0.5, device=DEV))
    with pytest.raises(RuntimeError, match="residual_scale"):
        fused_post_norm(t["x"], t["r"], residual_scale=p)
    with pytest.raises(RuntimeError, match="eps"):
        fused_pre_norm(t["x"], t["w"], eps=p)
    with fw.dual_level(), pytest.raises(RuntimeError, match="residual_scale"):
        fused_post_norm(t["x"], t["r"], residual_scale=fw.make_dual(torch.tensor(0.5), torch.tensor(1.0)))
    with torch.no_grad():
        assert torch.equal(fused_post_norm(t["x"], t["r"], residual_scale=p), fused_post_norm(t["x"], t["r"], residual_scale=0.5))


def test_saved_tensors_may_be_moved_or_made_again():
    """torch's hooks on saved tensors: kept on the host, or recomputed by a checkpoint."""
    from torch.utils.checkpoint import checkpoint
    t = _tensors()
    x, w, logits = (t[k].clone().requires_grad_(True) for k in ("x", "w", "logits"))

    def f(x, w, logits):
        n, h = fused_pre_norm(x, w, residual=t["r"])
        o = fused_router(logits, 3)
        return (fused_post_norm(n, h, w, gate=t["g"], residual_scale=0.5) * t["r"]).sum() + (o.topk_weights * t["r"][:, :3]).sum() + o.balance_loss + o.z_loss

    want = torch.autograd.grad(f(x, w, logits), [x, w, logits])
    with torch.autograd.graph.save_on_cpu():
        loss = f(x, w, logits)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, [x, w, logits]), want))
    loss = checkpoint(f, x, w, logits, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, [x, w, logits]), want))
