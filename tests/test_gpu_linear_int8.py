"""GPU tier: the W8A8 linear layer and its token quantiser against the 64-bit oracle.

The quantiser has to be exact.  The layer's sums of products are exact, so what is left per value is (float)acc, two products and
the sum with the bias, at most 4 roundings of 2^-24, and one rounding to the output type."""
import pytest
import torch

from oracle import dense_oracle as orc
from pyhip_b200 import int8_status, linear_int8, quantize_int8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _bound(y64, size, dtype):
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133          # half of the smallest subnormal, and some
    return torch.finfo(dtype).eps / 2 * y64.abs() + 4 * U * size * (1 + torch.finfo(dtype).eps) + tiny


def _check(y, y64, size):
    off = (y.double() - y64).abs() - _bound(y64, size, y.dtype)
    assert torch.isfinite(y).all() and float(off.max()) <= 0, f"{int((off > 0).sum())} of {off.numel()} values out of bounds, worst {float(off.max()):.3e}"


def _weight(N, K, seed, full=True):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    if full:
        w[:, 0], w[0] = -128, 127
    return w.to(DEV), (torch.rand(N, generator=g) * 0.01 + 1e-4).to(DEV)


def _equal(x):
    q, s = quantize_int8(x)
    q64, s64 = orc.quantize_int8(x)
    assert torch.equal(s.isnan(), s64.isnan()) and torch.equal(s.nan_to_num(), s64.nan_to_num())
    assert torch.equal(q.double(), q64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,K", [(1, 1), (3, 7), (5, 16), (130, 1040), (33, 2880), (9, 4099), (4, 16384), (2, 16383)])
def test_quantiser_is_exact(T, K, dtype):
    g = torch.Generator().manual_seed(T * 100 + K)
    _equal((torch.randn(T, K, generator=g) * 3).to(dtype).to(DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,K", [(593, 512), (700, 1040), (2000, 2880), (600, 16384), (600, 15)])
def test_quantiser_is_exact_for_many_rows(T, K, dtype):
    g = torch.Generator().manual_seed(T + K)
    x = torch.randn(T, K, generator=g) * torch.logspace(-30, 30, T)[:, None].clamp(1e-4 if dtype == torch.float16 else 0, 1e3 if dtype == torch.float16 else 1e31)
    x[3], x[4, 5], x[5, 6], x[-1, -1] = 0, float("inf"), float("nan"), float("-inf")
    half = (torch.arange(K) % 254 - 126.5).roll(1)
    x[7], x[8] = half, half * 3 * 2 ** -4                  # ties, exactly, where the row's largest value is 127 scales
    x[7, 0], x[8, 0] = 127, 127 * 3 * 2 ** -4
    x = x.to(dtype).to(DEV)
    _equal(x)
    _equal(torch.cat([x, x], dim=1)[:, 8:K + 8] if K % 8 == 0 else x)


def test_quantiser_at_the_borders():
    """Rows whose quotients are ties (scale a power of two, or 3 times one, which is exact in fp16), next to ties, zeros, tiny,
    subnormal and huge values, infinities and NaN."""
    half = torch.arange(-126, 127, dtype=torch.float32) + 0.5
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        for s in (1.0, 0.25, 3.0 * 2 ** -6):
            x = torch.cat([half, torch.tensor([127.0])]) * s
            x = x.to(dtype).to(DEV)
            _equal(torch.stack([x, -x]))
    near = torch.cat([torch.nextafter(half, torch.tensor(0.0)), torch.nextafter(half, torch.tensor(1e9)), torch.tensor([127.0])])
    for s in (1.0, 0.0123, 7.7e-9):
        _equal((near * s).to(DEV)[None])
    x = torch.randn(8, 64)
    x[1] = 0
    x[2] *= 1e-38
    x[3] *= 1e-42
    x[4, 5] = float("inf")
    x[5, 6] = float("nan")
    x[6, 7], x[6, 8] = float("-inf"), float("nan")
    x[7] *= 1e36
    _equal(x.to(DEV))
    _equal(x.to(torch.bfloat16).to(DEV))


def test_quantiser_reads_strided_rows_and_any_shape():
    x = torch.randn(4, 6, 100, device=DEV, dtype=torch.bfloat16)
    _equal(x)
    wide = torch.randn(9, 333, device=DEV, dtype=torch.float16)
    _equal(wide[:, 5:205])
    _equal(wide[::2, 8:264])
    _equal(wide.t()[:64])
    _equal(wide[:1].expand(5, 333))
    _equal(wide[0])
    q, s = quantize_int8(wide[:0])
    assert q.shape == (0, 333) and s.shape == (0,)


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("T,N,K", [(1, 1, 16), (1, 130, 144), (2, 128, 2880), (16, 256, 128), (17, 1001, 1040), (64, 2880, 512),
                                   (127, 8, 4096), (129, 136, 16), (256, 300, 640), (333, 1001, 1040), (300, 512, 7168), (1000, 2048, 7168), (700, 1501, 4096), (1000, 2043, 4096), (2049, 2311, 272)])
def test_layer_matches_64_bits(T, N, K, variant):
    g = torch.Generator().manual_seed(T + N + K)
    w, ws = _weight(N, K, T + N)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16).to(DEV)
    y64, size = orc.linear_int8(*orc.quantize_int8(x), w, ws)
    _check(linear_int8(x, w, ws, variant=variant), y64, size)
    assert int8_status(DEV) == (0, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,N,K", [(1, 2880, 2880), (1, 129, 16384), (8, 300, 4096), (3, 2880, 2896), (5, 14336, 2048), (8, 64, 16), (9, 64, 4096), (2, 40, 8208)])
def test_few_tokens(T, N, K, dtype):
    """One token, which the split kernel quantises itself, and a few: rows on and off the 16-byte grid, apart from one another,
    the last ones of a buffer."""
    g = torch.Generator().manual_seed(T * K)
    w, ws = _weight(N, K, T)
    wide = torch.randn(T, K + 24, generator=g).to(dtype).to(DEV)
    for x in (wide[:, :K].contiguous(), wide[:, 8:K + 8], wide[:, 3:K + 3], wide[:, 24:]):
        y = linear_int8(x, w, ws, out_dtype=torch.bfloat16)
        _check(y, *orc.linear_int8(*orc.quantize_int8(x), w, ws))
        q, s = quantize_int8(x)
        assert torch.equal(y, linear_int8(q, w, ws, x_scale=s, out_dtype=torch.bfloat16))
    assert int8_status(DEV) == (0, 0)


@pytest.mark.parametrize("T,N,K", [(4, 64, 16), (600, 264, 1040), (2000, 1160, 512), (5000, 515, 256)])
def test_layer_types_bias_and_prequantised_rows(T, N, K):
    g = torch.Generator().manual_seed(T)
    w, ws = _weight(N, K, N)
    bias = torch.randn(N, generator=g).to(DEV)
    x = torch.randn(T, K, generator=g)
    for dtype, out in ((torch.float16, None), (torch.float32, torch.float16), (torch.bfloat16, torch.float16)):
        xd = (x * 0.01).to(dtype).to(DEV)
        y = linear_int8(xd, w, ws * 0.1, bias=bias, out_dtype=out)
        assert y.dtype == torch.float16
        _check(y, *orc.linear_int8(*orc.quantize_int8(xd), w, ws * 0.1, bias))
    q, s = quantize_int8(x.to(DEV))
    y = linear_int8(q, w, ws, x_scale=s, bias=bias)
    assert y.dtype == torch.bfloat16
    _check(y, *orc.linear_int8(q, s, w, ws, bias))


def test_largest_sums_are_exact():
    """-128 * -128 over the longest K that fits int32."""
    K = (1 << 17) - 16
    q = torch.full((3, K), -128, dtype=torch.int8, device=DEV)
    w = torch.full((5, K), -128, dtype=torch.int8, device=DEV)
    w[1:] = 127
    one = torch.ones(5, device=DEV)
    for variant in (1, 2):
        y = linear_int8(q, w, one, x_scale=torch.ones(3, device=DEV), variant=variant)
        _check(y, *orc.linear_int8(q, torch.ones(3, device=DEV), w, one))


def test_layer_shapes_strides_and_empty_batches():
    w, ws = _weight(48, 64, 3)
    x = torch.randn(3, 5, 64, device=DEV, dtype=torch.bfloat16)
    y = linear_int8(x, w, ws)
    assert y.shape == (3, 5, 48)
    flat = linear_int8(x.reshape(15, 64), w, ws)
    assert torch.equal(y.reshape(15, 48), flat)
    assert linear_int8(x[0, 0], w, ws).shape == (48,)
    assert linear_int8(x[:0], w, ws).shape == (0, 5, 48)
    wide = torch.randn(70, 200, device=DEV, dtype=torch.bfloat16)
    assert torch.equal(linear_int8(wide[:, 3:67], w, ws), linear_int8(wide[:, 3:67].contiguous(), w, ws))
    q, s = quantize_int8(wide[:, :65])
    assert torch.equal(linear_int8(q[:, 1:], w, ws, x_scale=s), linear_int8(q[:, 1:].clone(), w, ws, x_scale=s))
    odd = torch.empty(48 * 64 + 1, dtype=torch.int8, device=DEV)[1:].view(48, 64).copy_(w)      # a weight off the 16-byte grid
    assert torch.equal(linear_int8(x, odd, ws), y)
    assert torch.equal(linear_int8(x, w.t().contiguous().t(), ws), y)


def test_rows_that_hold_infinities_stay_their_own():
    w, ws = _weight(40, 64, 5)
    for T in (6, 700):
        x = torch.randn(T, 64, device=DEV, dtype=torch.bfloat16)
        good = linear_int8(x, w, ws)
        x[2, 3], x[4, 5] = float("inf"), float("nan")
        y = linear_int8(x, w, ws)
        keep = torch.ones(T, dtype=torch.bool, device=DEV)
        keep[2] = keep[4] = False
        assert torch.equal(y[keep], good[keep]) and y[~keep].isnan().all()


def test_one_row_of_zeros_infinities_and_tiny_values():
    w, ws = _weight(40, 128, 6)
    x = torch.randn(1, 128, device=DEV, dtype=torch.float32)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        zero = torch.zeros(1, 128, device=DEV, dtype=dtype)
        assert (linear_int8(zero, w, ws, out_dtype=torch.bfloat16) == 0).all()
        for bad in (float("inf"), float("nan"), float("-inf")):
            y = x.to(dtype).clone()
            y[0, 77] = bad
            assert linear_int8(y, w, ws, out_dtype=torch.bfloat16).isnan().all()
        tiny = (x * 1e-6).to(dtype)
        _check(linear_int8(tiny, w, ws, out_dtype=torch.bfloat16), *orc.linear_int8(*orc.quantize_int8(tiny), w, ws))


@pytest.mark.parametrize("T", [3, 900])
def test_rows_behind_the_output_are_left_alone(T):
    """The output's neighbours in memory: a layer call must not write outside its rows, whichever way they are stored."""
    for N in (40, 43, 1001):
        w, ws = _weight(N, 64, N)
        x = torch.randn(T, 64, device=DEV, dtype=torch.bfloat16)
        want = linear_int8(x, w, ws)
        from pyhip_b200 import _lib
        pad = 8192
        buf = torch.full((T * N + 2 * pad,), 777.0, dtype=torch.bfloat16, device=DEV)
        y = buf[pad:pad + T * N]
        ws_bytes = (T * 64 + 255) // 256 * 256 + 4 * T
        scratch = torch.empty(ws_bytes, dtype=torch.uint8, device=DEV)
        _lib.check(_lib.lib().b200moe_linear_int8(x.data_ptr(), 64, _lib.T_BF16, None, w.data_ptr(), ws.data_ptr(), None, T, N, 64,
                                                  _lib.T_BF16, 0, scratch.data_ptr(), ws_bytes, None, y.data_ptr(),
                                                  torch.cuda.current_stream().cuda_stream), "linear_int8")
        assert torch.equal(y.view(T, N), want)
        assert (buf[:pad] == 777).all() and (buf[pad + T * N:] == 777).all()


@pytest.mark.parametrize("T", [1, 40, 600])
def test_graph_replay_and_streams(T):
    w, ws = _weight(264, 512, T)
    x = torch.randn(T, 512, device=DEV, dtype=torch.bfloat16)
    want = linear_int8(x, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [linear_int8(x, w, ws) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in ys)
    x2 = x.clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        a = linear_int8(x2, w, ws)
    with torch.cuda.graph(g2):
        b = linear_int8(x2, w, ws)
    other = torch.randn_like(x)
    for src in (x, other, x):
        x2.copy_(src)
        a.zero_(), b.zero_()
        g1.replay(), g2.replay(), g1.replay()
        torch.cuda.synchronize()
        ref = linear_int8(src, w, ws)
        assert torch.equal(a, ref) and torch.equal(b, ref)


def test_weights_written_just_before_the_call_are_seen():
    """The split kernel fetches weights while the quantiser still runs: a weight that the stream writes right in front has to
    arrive, also where the launches chain back to back."""
    w, ws = _weight(2880, 2880, 1)
    x = torch.randn(4, 2880, device=DEV, dtype=torch.bfloat16)
    for i in range(20):
        w.random_(-127, 128)
        y = linear_int8(x, w, ws)
        if i % 5 == 0:
            _check(y, *orc.linear_int8(*orc.quantize_int8(x), w, ws))
        src = torch.randn(2880, 2880, device=DEV, dtype=torch.bfloat16)
        q, s = quantize_int8(src)
        y = linear_int8(x, q, s)
        if i % 5 == 0:
            _check(y, *orc.linear_int8(*orc.quantize_int8(x), q, s))


def test_layer_refuses_what_it_cannot_do():
    w, ws = _weight(32, 64, 2)
    x = torch.randn(4, 64, device=DEV, dtype=torch.bfloat16)
    q, s = quantize_int8(x)
    for call in (lambda: linear_int8(x[:, :48], w, ws), lambda: linear_int8(x, w[:, :40], ws), lambda: linear_int8(x, w, ws[:5]),
                 lambda: linear_int8(x[:, :8], w[:, :8], ws), lambda: linear_int8(q, w, ws), lambda: linear_int8(q, w, ws, x_scale=s[:2]),
                 lambda: linear_int8(x, w, ws, x_scale=s), lambda: linear_int8(x, w, ws, bias=ws[:3]), lambda: linear_int8(x, w, ws, variant=3),
                 lambda: linear_int8(x, w.cpu(), ws), lambda: quantize_int8(torch.empty(2, 0, device=DEV)),
                 lambda: quantize_int8(torch.empty(1, 16385, device=DEV))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: linear_int8(x, w.float(), ws), lambda: linear_int8(x.double(), w, ws),
                 lambda: linear_int8(x, w, ws, out_dtype=torch.float32), lambda: quantize_int8(q)):
        with pytest.raises(TypeError):
            call()
    x.requires_grad_(True)
    for call in (lambda: linear_int8(x, w, ws), lambda: quantize_int8(x)):
        with pytest.raises(RuntimeError):
            call()
    with torch.no_grad():
        linear_int8(x, w, ws)
