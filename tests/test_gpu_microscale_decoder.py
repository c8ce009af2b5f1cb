"""The decoder with microscaled projections and with experts (apsi_b200.decoder), against the same network with every
product taken in float64 over the values the operands stand for."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
SMALL = dict(H=256, L=2, nh=4, kvh=2, dh=64, I=480, V=1000)


def rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


@pytest.fixture
def slow(monkeypatch):
    """Products in float64 from the quantised operands, rounded once."""
    from apsi_b200 import microscale as mx

    def finish(y, bias, out, accumulate):
        y = y if bias is None else y + bias.double()
        if out is None:
            return y.to(torch.bfloat16)
        out.copy_((y + out.double() if accumulate else y).to(torch.bfloat16))
        return out

    def linear(x, w, bias=None, out=None, accumulate=False, tensor_scale=None):
        q = x if isinstance(x, mx.MxTensor) else mx.quantize(x, w.fmt, tensor_scale)
        return finish(q.dequantize().double() @ w.dequantize().double().T, bias, out, accumulate)

    def grouped(x, w, bias=None, out=None, accumulate=False):
        xv, wv, at = x.dequantize().double(), w.dequantize().double(), x.offsets.tolist()
        return finish(torch.cat([xv[at[e]:at[e + 1]] @ wv[e].T for e in range(len(at) - 1)]), bias, out, accumulate)

    def use():
        monkeypatch.setattr(mx, "linear", linear)
        monkeypatch.setattr(mx, "linear_grouped", grouped)
    return use


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("experts", [0, 6])
def test_prefill_matches_float64_products(cuda, slow, fmt, experts):
    """Both sides round each product to bfloat16 (unit roundoff 2^-8) from sums that agree to float32's error, so only
    roundings on a boundary differ, and what they move: a code of the next quantisation now and then.  Held to the
    decoder's bar for its other formats, 3e-2."""
    from apsi_b200.decoder import DecoderConfig, QuantDecoder
    model = QuantDecoder(DecoderConfig(**SMALL, E=experts, topk=2), device=cuda, fmt=fmt, seed=3)
    ids = torch.randint(0, SMALL["V"], (3, 50), device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    got = model.prefill(ids, model.new_cache(3, 64))
    slow()
    assert rel(got, model.prefill(ids, model.new_cache(3, 64))) < 3e-2


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("experts", [0, 6])
def test_generation_through_a_graph(cuda, fmt, experts):
    from apsi_b200 import kernels
    from apsi_b200.decoder import DecoderConfig, QuantDecoder
    model = QuantDecoder(DecoderConfig(**SMALL, E=experts, topk=2), device=cuda, fmt=fmt, seed=4)
    ids = torch.randint(0, SMALL["V"], (2, 8), device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))
    a, _ = model.generate(ids, 6, graph=True)
    b, _ = model.generate(ids, 6, graph=False)
    assert torch.equal(a, b)
    assert kernels.device_errors(cuda) == 0
    assert model.weight_bytes() > 0


def test_experts_need_a_microscaled_format(cuda):
    from apsi_b200._lib import LowbitError
    from apsi_b200.decoder import DecoderConfig, QuantDecoder
    with pytest.raises(LowbitError):
        QuantDecoder(DecoderConfig(**SMALL, E=4), device=cuda, fmt="int4")
