"""GPU tier: kernels that hold tensor memory side by side -- the W8A8 layer in its split-K and its pair form, the MoE layer and torch's own
products on streams of their own -- and the dense operators called from several host threads.  Results are those of the calls
made alone, bit for bit."""
import threading

import pytest
import torch

from pyhip_b200 import QuantType, fused_moe, fused_post_norm, fused_pre_norm, fused_router, int8_status, linear_int8, quantize_int8, synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_tensor_memory_kernels_on_several_streams():
    H, I, E, K, T = 512, 1024, 8, 2, 1024
    w1, s1, w2, s2 = (t.to(DEV) for t in synth.make_weights_mxfp4(E, H, I, seed=1))
    x = synth.make_hidden(T, H, 2).to(DEV)
    tw, ids = (t.to(DEV) for t in synth.make_routing(T, E, K))
    w, ws = quantize_int8(torch.randn(4096, H, device=DEV))
    a = torch.randn(2048, 512, device=DEV, dtype=torch.bfloat16)
    few, many = x[:64].contiguous(), x[:900].contiguous()
    calls = [lambda: fused_moe(x, w1, w2, tw, ids, quant_type=QuantType.per_1x32, w1_scale=s1, w2_scale=s2),
             lambda: linear_int8(few, w, ws), lambda: linear_int8(x[:1], w, ws), lambda: linear_int8(many, w, ws), lambda: a @ a.t()]
    want = [c().clone() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    torch.cuda.synchronize()
    for _ in range(40):
        for c, s, g in zip(calls, streams, got):
            with torch.cuda.stream(s):
                g.append(c())
    torch.cuda.synchronize()
    for k, (g, r) in enumerate(zip(got, want)):
        assert all(torch.equal(v, r) for v in g), k
    assert int8_status(DEV) == (0, 0)


def test_operators_from_several_host_threads():
    def make(seed):
        g = torch.Generator().manual_seed(seed)
        t = {k: torch.randn(*s, generator=g).to(DEV) for k, s in dict(x=(70, 512), r=(70, 512), w=(512,), logits=(70, 32)).items()}
        t["iw"], t["ws"] = quantize_int8(torch.randn(256, 512, generator=g).to(DEV))
        return t

    def step(t):
        x, w, logits = (t[k].detach().clone().requires_grad_(True) for k in ("x", "w", "logits"))
        h, n = fused_post_norm(x, t["r"], w, next_weight=w)
        o = fused_router(logits, 4)
        grads = torch.autograd.grad([h, n, o.topk_weights, o.balance_loss], [x, w, logits], [t["r"], t["r"], torch.ones_like(o.topk_weights),
                                                                                             torch.ones_like(o.balance_loss)])
        with torch.no_grad():
            q, s, _ = fused_pre_norm(t["x"], t["w"], residual=t["r"], quant="int8")
            y = linear_int8(q, t["iw"], t["ws"], x_scale=s), linear_int8(t["x"][:1], t["iw"], t["ws"])
        return [v.detach() for v in (h, n, *o, *grads, *y)]

    data = [make(k) for k in range(4)]
    want = [step(t) for t in data]
    torch.cuda.synchronize()
    wrong, failed = [], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(25):
                    got = step(data[k])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                        wrong.append(k)
        except Exception as e:                               # noqa: BLE001  (told below)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=120)
    assert not failed and not wrong and not any(t.is_alive() for t in threads), (failed, wrong)
