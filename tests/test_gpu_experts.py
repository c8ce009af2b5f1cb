"""Routing, combine and the expert MLP on the GPU, against float64 oracles."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import microscale as ora  # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ex(cuda):
    from apsi_b200 import experts
    return experts


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def check_route(r, logits, k, normalize):
    w, chosen, offsets, rows, slots = ora.route(f64(logits), k, normalize)
    assert np.array_equal(r.experts.cpu().numpy(), chosen)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    assert np.array_equal(r.rows.cpu().numpy(), rows)
    assert np.array_equal(r.slots.cpu().numpy(), slots)
    # expf within 2 units in the last place, a sum of E and a quotient in float32
    assert np.allclose(f64(r.weights), w, rtol=(logits.shape[1] + 8) * 2.0 ** -24, atol=2.0 ** -100)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 33, 32), (16, 64, 8), (65, 31, 4), (64, 32, 1), (300, 128, 10),
                                   (1000, 257, 3), (129, 1024, 32), (5000, 7, 7)])
def test_route(ex, dtype, normalize, T, E, k):
    g = np.random.default_rng(T + E)
    lg = torch.from_numpy(g.standard_normal((T, E)).astype(np.float32) * 2).cuda().to(DT[dtype])
    check_route(ex.route(lg, k, normalize), lg, k, normalize)


def test_route_ties_masks_and_non_numbers(ex):
    inf, nan = float("inf"), float("nan")
    lg = torch.tensor([[0.0, -0.0, 0.0, 0.0], [1, 2, 2, 1], [-inf, -inf, 3, -inf], [-inf] * 4, [nan] * 4, [nan, 1, -inf, nan],
                       [inf, 0, inf, 5], [-1e38, 1e38, 0, 1e-38], [88.0, -88.0, 0.0, 200.0]], device="cuda")
    for k in (1, 2, 4):
        for normalize in (True, False):
            r = ex.route(lg, k, normalize)
            check_route(r, lg, k, normalize)
            assert torch.isfinite(r.weights).all()


def test_route_strided_and_empty(ex):
    big = torch.randn((50, 40), device="cuda")
    check_route(ex.route(big[::2, 3:30], 2), big[::2, 3:30], 2, True)
    r = ex.route(torch.empty((0, 8), device="cuda"), 2)
    assert r.offsets.tolist() == [0] * 9 and r.rows.numel() == 0 and r.slots.shape == (0, 2)


@pytest.mark.parametrize("T,k,H", [(1, 1, 1), (3, 2, 7), (16, 8, 2048), (100, 5, 1000), (77, 1, 33), (300, 32, 64), (4, 9, 4096)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_combine(ex, T, k, H, accumulate):
    z = torch.randn((T * k + 3, H), device="cuda").to(torch.bfloat16)
    slots = torch.randperm(T * k, device="cuda").to(torch.int32).view(T, k)
    w = torch.softmax(torch.randn((T, k), device="cuda"), 1)
    if k > 1:
        w[0, 0] = 0                                     # a weight of 0 adds nothing, whatever z holds
        z[slots[0, 0].long()] = float("nan")
    out = torch.randn((T, H), device="cuda").to(torch.bfloat16) if accumulate else None
    before = f64(out) if accumulate else 0.0
    zz = torch.where(torch.isnan(z), torch.zeros_like(z), z)
    ref = ora.combine(f64(zz), f64(w), slots.cpu().numpy()) + before
    mass = ora.combine(np.abs(f64(zz)), f64(w), slots.cpu().numpy()) + np.abs(before)
    y = ex.combine(z, w, slots, out=out, accumulate=accumulate)
    err = (k + 1) * 2.0 ** -24 * mass
    lo, hi = (torch.from_numpy(ref + s * err).float().to(torch.bfloat16).double().numpy() for s in (-1, 1))
    assert ((lo <= f64(y)) & (f64(y) <= hi)).all()


def test_combine_strides_and_bad_slots(ex):
    from apsi_b200 import kernels, _lib
    kernels.device_errors()
    z = torch.randn((8, 40), device="cuda").to(torch.bfloat16)
    w = torch.full((3, 2), 0.5, device="cuda")
    slots = torch.tensor([[0, 1], [2, 8], [-1, 5]], dtype=torch.int32, device="cuda")
    y = ex.combine(z[:, 1:34], w, slots)
    want = torch.stack([(z[0, 1:34].float() + z[1, 1:34].float()) / 2, z[2, 1:34].float() / 2, z[5, 1:34].float() / 2])
    assert torch.equal(y, want.to(torch.bfloat16))
    assert kernels.device_errors() == _lib.DEVERR_BAD_INDEX


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("T", [1, 5, 200])
def test_expert_mlp(ex, fmt, T):
    """The layer equals its parts put together by hand in float64 from the same quantised operands; the hidden
    activations are taken from the run, since a rounding of theirs may move a code."""
    from apsi_b200 import kernels, microscale as mx
    E, H, I, k = 6, 256, 160, 2
    g = torch.Generator(device="cuda").manual_seed(T)
    router, gu, down = (torch.randn(s, generator=g, device="cuda") * 0.08 for s in ((E, H), (E, 2 * I, H), (E, H, I)))
    x = torch.randn((T, H), generator=g, device="cuda").to(torch.bfloat16)
    mlp = ex.ExpertMLP(router, gu, down, k, fmt)
    y = mlp(x)
    r = ex.route(torch.matmul(x, mlp.router.t()), k)
    q = mx.quantize(x, fmt, rows=r.rows, offsets=r.offsets)
    h = kernels.act_mul(mx.linear_grouped(q, mlp.gate_up), I, 0)
    hq = mx.quantize(h, fmt, offsets=r.offsets).dequantize().double()
    dn, off = mlp.down.dequantize().double(), r.offsets.tolist()
    z = torch.cat([hq[off[e]:off[e + 1]] @ dn[e].T for e in range(E)])
    want = (z[r.slots.long()] * r.weights.double()[..., None]).sum(1)
    # z is rounded to bfloat16 (unit roundoff 2^-8), weighted by at most 1 in all, and the sum rounded once more
    bound = 2.0 ** -8 * ((z.abs()[r.slots.long()] * r.weights.double()[..., None]).sum(1) + want.abs()) * 1.02 + 1e-6
    assert ((y.double() - want).abs() <= bound).all()
    res = torch.randn((T, H), device="cuda").to(torch.bfloat16)
    out = res.clone()
    assert mlp(x, out=out, accumulate=True) is out
    assert ((out.double() - res.double() - want).abs() <= bound + 2.0 ** -8 * (res.double().abs() + want.abs())).all()


def test_expert_mlp_without_tokens(ex):
    E, H, I = 3, 64, 32
    mlp = ex.ExpertMLP(torch.randn((E, H), device="cuda"), torch.randn((E, 2 * I, H), device="cuda"),
                       torch.randn((E, H, I), device="cuda"), 1)
    assert mlp(torch.empty((0, H), device="cuda", dtype=torch.bfloat16)).shape == (0, H)


def test_refusals(ex):
    from apsi_b200._lib import LowbitError
    lg = torch.randn((4, 8), device="cuda")
    z = torch.randn((8, 16), device="cuda").to(torch.bfloat16)
    w, s = torch.ones((4, 2), device="cuda"), torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    bad = [lambda: ex.route(lg.cpu(), 2), lambda: ex.route(lg.double(), 2), lambda: ex.route(lg[0], 2), lambda: ex.route(lg, 0),
           lambda: ex.route(lg, 9), lambda: ex.route(torch.randn((2, 40), device="cuda"), 33), lambda: ex.route(lg.t(), 2),
           lambda: ex.route(torch.randn((1, 1025), device="cuda"), 1), lambda: ex.combine(z.float(), w, s),
           lambda: ex.combine(z, w, s.long()), lambda: ex.combine(z, w.to(torch.bfloat16), s), lambda: ex.combine(z, w, s[:, :1]),
           lambda: ex.combine(z, w[:, :0], s[:, :0]), lambda: ex.combine(z.cpu(), w, s), lambda: ex.combine(z, w, s, accumulate=True),
           lambda: ex.combine(z, w, s, out=z[:3]), lambda: ex.ExpertMLP(torch.randn((2, 64), device="cuda"),
                                                                        torch.randn((2, 64, 64), device="cuda"),
                                                                        torch.randn((2, 64, 64), device="cuda"), 1)]
    for i, f in enumerate(bad):
        with pytest.raises(LowbitError):
            f()
            pytest.fail(f"case {i} was taken")
