"""Microscaled 4-bit floats on the GPU: quantise, dequantise, products, products by expert, against float64 oracles."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import microscale as ora  # noqa: E402

pytestmark = pytest.mark.gpu
FMTS = ["mxfp4", "nvfp4"]
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def mx(cuda):
    from apsi_b200 import microscale
    return microscale


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def codes_of(q):
    c = q.codes.cpu().numpy()
    return np.stack((c & 15, c >> 4), -1).reshape(c.shape[0], -1)


def acts(seed, R, K, dtype=torch.bfloat16, spread=1.0):
    g = np.random.default_rng(seed)
    x = g.standard_normal((R, K)) * np.exp(spread * g.standard_normal((R, 1)))
    return torch.from_numpy(x.astype(np.float32)).cuda().to(dtype)


def sum_error(mass, K):
    """What a float32 sum may be off: each instruction adds 64 products to the accumulator, and both the sum inside and the
    addition lose at most 2^-22 of what they add up."""
    return (K / 64 + 2) * 2.0 ** -22 * mass + 1e-30


def assert_rounds(y, ref, err):
    """y is the bfloat16 rounding of some value within err of ref (rounding is monotone, so no slack is needed for it)."""
    lo, hi = (torch.from_numpy(ref + s * err).to(torch.float32).to(torch.bfloat16).double().numpy() for s in (-1, 1))
    got = f64(y)
    assert ((lo <= got) & (got <= hi)).all(), np.abs(got - ref).max()


# ------------------------------------------------------------------------------------------------ quantise
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,K", [(1, 1), (1, 4096), (3, 31), (5, 33), (130, 257), (257, 640), (2, 11008), (64, 1000)])
def test_quantize_is_exact(mx, fmt, dtype, R, K):
    x = acts(R * K, R, K, DT[dtype])
    t = 2.0 ** -3
    q = mx.quantize(x, fmt, tensor_scale=t if fmt == "nvfp4" else None)
    code, byte, val = ora.quantize(f64(x), fmt, t)
    got = codes_of(q)
    assert np.array_equal(got[:, :K], code[:, :K])
    assert not got[:, K:].any()
    assert np.array_equal(mx.plain_scales(q).cpu().numpy(), byte[:, :-(-K // ora.BLOCK[fmt])])
    assert np.array_equal(f64(mx.dequantize(q)), val)
    for d in (torch.bfloat16, torch.float16):
        want = torch.from_numpy(val).to(torch.float32).to(d)
        assert np.array_equal(f64(mx.dequantize(q, d)), f64(want))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_ties_and_edges(mx, fmt):
    """Every midpoint and its neighbours, saturation, tiny and huge blocks, zeros and signed zeros."""
    mids = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5], np.float32)
    rows = []
    for s in (1.0, 2.0 ** 60, 2.0 ** -100, 2.0 ** -126):
        near = np.concatenate([mids, np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(9))]) * np.float32(s)
        row = np.zeros(64, np.float32)
        row[:near.size] = near * np.where(np.arange(near.size) % 2, -1, 1)
        row[30], row[31], row[63] = 6 * s, -0.0, 7.5 * s
        row[15] = row[47] = 6 * s
        rows.append(row)
    rows.append(np.zeros(64, np.float32))
    rows.append(np.full(64, np.finfo(np.float32).max))
    rows.append(np.full(64, np.float32(1e-45)))
    x = np.stack(rows)
    q = mx.quantize(torch.from_numpy(x).cuda(), fmt, tensor_scale=1.0 if fmt == "nvfp4" else None)
    code, byte, val = ora.quantize(x, fmt)
    assert np.array_equal(codes_of(q), code)
    assert np.array_equal(mx.plain_scales(q).cpu().numpy(), byte)
    assert np.array_equal(f64(q.dequantize()), val.astype(np.float32).astype(np.float64))


def test_every_e4m3_step_and_a_scale_that_is_no_power_of_two(mx):
    g = np.random.default_rng(5)
    x = (g.standard_normal((64, 512)) * np.exp2(g.integers(-14, 14, (64, 32))).repeat(16, 1)).astype(np.float32)
    for t in (1.0, 0.0371, 2.0 ** -120):
        t = float(np.float32(t))
        q = mx.quantize(torch.from_numpy(x).cuda(), "nvfp4", tensor_scale=torch.tensor([t], device="cuda"))
        with np.errstate(over="ignore"):
            code, byte, _ = ora.quantize(x, "nvfp4", t)
        assert np.array_equal(mx.plain_scales(q).cpu().numpy(), byte)
        assert np.array_equal(codes_of(q), code)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_no_number_stands_for_nans(mx, fmt, bad):
    x = torch.ones((2, 96), device="cuda")
    x[1, 40] = bad
    v = mx.quantize(x, fmt, tensor_scale=1.0 if fmt == "nvfp4" else None).dequantize()
    lost = torch.zeros_like(x, dtype=torch.bool)
    lost[1, (32 if fmt == "mxfp4" else 32):(64 if fmt == "mxfp4" else 48)] = True
    assert torch.equal(torch.isnan(v), lost)
    want = ora.quantize(f64(x), fmt)[2]
    assert np.array_equal(f64(v)[~lost.cpu().numpy()], want[~lost.cpu().numpy()])


@pytest.mark.parametrize("dtype", list(DT))
def test_the_tensor_scale_is_found(mx, dtype):
    for scale in (1e-30 if dtype == "f32" else 1e-3, 1.0, 77.0, 5e3):
        x = (acts(3, 70, 1030, torch.float32, 0.5) * scale).to(DT[dtype])
        x[0, 0] = float("nan")
        q = mx.quantize(x, "nvfp4")
        assert float(q.tensor_scale) == ora.auto_scale(f64(x))
    assert float(mx.quantize(torch.zeros((3, 40), device="cuda", dtype=DT[dtype]), "nvfp4").tensor_scale) == 1.0
    x = torch.full((1, 16), 2688.0, device="cuda", dtype=DT[dtype])           # exactly the top of the range
    assert float(mx.quantize(x, "nvfp4").tensor_scale) == 1.0


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_with_a_stride_and_off_alignment(mx, fmt):
    big = acts(1, 40, 301)
    t = 0.25 if fmt == "nvfp4" else None
    for x in (big[:, 3:300], big[::3, :128], big[:, 1:2], big[7:8]):
        want = ora.quantize(f64(x), fmt, 0.25)[2]
        assert np.array_equal(f64(mx.quantize(x, fmt, tensor_scale=t).dequantize()), want)


@pytest.mark.parametrize("fmt", FMTS)
def test_gathered_rows_in_ragged_groups(mx, fmt):
    x = acts(9, 50, 200)
    sizes = [0, 1, 127, 0, 128, 129, 0, 3, 0]
    offsets = torch.tensor(np.concatenate(([0], np.cumsum(sizes))), dtype=torch.int32, device="cuda")
    rows = torch.randint(0, 50, (sum(sizes),), device="cuda", dtype=torch.int32)
    t = 0.25 if fmt == "nvfp4" else None
    q = mx.quantize(x, fmt, tensor_scale=t, rows=rows, offsets=offsets)
    assert np.array_equal(f64(q.dequantize()), ora.quantize(f64(x[rows.long()]), fmt, 0.25)[2])


@pytest.mark.parametrize("fmt", FMTS)
def test_expert_matrices_and_checkpoint_arrays(mx, fmt):
    W = acts(4, 3 * 70, 96, torch.float32).view(3, 70, 96)
    t = 0.25 if fmt == "nvfp4" else None
    q = mx.quantize(W, fmt, tensor_scale=t)
    val = ora.quantize(f64(W).reshape(210, 96), fmt, 0.25)[2].reshape(3, 70, 96)
    assert np.array_equal(f64(q.dequantize()), val)
    s = mx.plain_scales(q)
    again = mx.pack(q.codes.view(3, 70, 48), s, 96, fmt, tensor_scale=t)
    assert np.array_equal(f64(again.dequantize()), val)
    # a K that is not whole blocks, and code bytes with something behind the last value
    one = mx.pack(q.codes.view(3, 70, 48)[1], s[1], 77, fmt, tensor_scale=t)
    assert np.array_equal(f64(one.dequantize()), val[1][:, :77])
    assert not codes_of(one)[:, 77:].any()


def test_row_indices_and_offsets_out_of_range_are_reported(mx):
    from apsi_b200 import kernels, _lib
    kernels.device_errors()
    x = acts(2, 8, 64)
    rows = torch.tensor([0, 8, 7, -1], dtype=torch.int32, device="cuda")
    v = mx.quantize(x, "mxfp4", rows=rows).dequantize()
    assert not v[1].any() and not v[3].any() and v[0].any()
    assert kernels.device_errors() == _lib.DEVERR_BAD_INDEX
    off = torch.tensor([0, 6, 3, 900], dtype=torch.int32, device="cuda")       # falls, then leaves the tensor
    q = mx.quantize(x, "mxfp4", offsets=off)
    w = mx.quantize(torch.randn((3, 16, 64), device="cuda"), "mxfp4")
    y = mx.linear_grouped(q, w)
    assert torch.isfinite(y).all()
    assert kernels.device_errors() == _lib.DEVERR_BAD_INDEX
    assert kernels.device_errors() == 0


# ------------------------------------------------------------------------------------------------ products
def product_case(mx, fmt, M, N, K, seed=0, **kw):
    x, w = acts(seed, M, K), acts(seed + 1, N, K, torch.float32, 0.3) * 0.05
    t = (0.25, 2.0 ** -12) if fmt == "nvfp4" else (None, None)
    q, p = mx.quantize(x, fmt, tensor_scale=t[0]), mx.quantize(w, fmt, tensor_scale=t[1])
    xv, wv = q.dequantize().double(), p.dequantize().double()
    return q, p, f64(xv @ wv.T), f64(xv.abs() @ wv.abs().T)


SHAPES = [(1, 128, 256), (1, 1, 32), (1, 17, 1), (2, 300, 31), (3, 257, 100), (16, 512, 1024), (17, 130, 288), (33, 4096, 4096),
          (64, 1000, 8192), (65, 256, 544), (100, 11008, 320), (128, 640, 2048), (129, 129, 129), (200, 333, 4096),
          (257, 513, 777), (300, 8200, 160), (1000, 4096, 96), (2048, 5000, 512), (1, 28672, 8192), (2300, 300, 64),
          (5, 600, 8448), (2, 100, 70000), (257, 20000, 512)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(mx, fmt, M, N, K):
    q, p, ref, mass = product_case(mx, fmt, M, N, K, seed=M + N + K)
    y = mx.linear(q, p)
    assert y.shape == (M, N) and y.dtype == torch.bfloat16
    assert_rounds(y, ref, sum_error(mass, K))
    assert torch.equal(y, mx.linear(q, p))                                     # the same bits every time


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (40, 257, 4096), (128, 100, 96), (200, 260, 300), (640, 8200, 256)])
def test_bias_accumulate_and_a_strided_output(mx, fmt, M, N, K):
    q, p, ref, mass = product_case(mx, fmt, M, N, K, seed=7)
    bias = torch.randn((N,), device="cuda").to(torch.bfloat16)
    for pad in (0, 1, 8):
        big = torch.randn((M, N + pad + 3), device="cuda").to(torch.bfloat16)
        for off in (0, 1):
            was = big.clone()
            y = big[:, off:off + N]
            before = f64(y)
            assert mx.linear(q, p, bias=bias, out=y, accumulate=True) is y
            want = ref + f64(bias) + before
            slack = 2.0 ** -23 * 4 * (np.abs(ref) + np.abs(f64(bias)) + np.abs(before))
            assert_rounds(y, want, sum_error(mass, K) + slack)
            was[:, off:off + N] = y
            assert torch.equal(was, big)                                       # nothing beside the output
    y = mx.linear(q, p, bias=bias)
    want = ref + f64(bias)
    assert_rounds(y, want, sum_error(mass, K) + 2.0 ** -21 * np.abs(want))


@pytest.mark.parametrize("fmt", FMTS)
def test_float_rows_are_quantised_on_the_way_in(mx, fmt):
    w = mx.quantize(acts(1, 96, 160, torch.float32), fmt)
    x = acts(2, 12, 160).view(3, 4, 160)
    y = mx.linear(x, w)
    assert y.shape == (3, 4, 96)
    assert torch.equal(y.view(12, 96), mx.linear(mx.quantize(x.view(12, 160), fmt), w))


@pytest.mark.parametrize("fmt", FMTS)
def test_nan_blocks_touch_their_own_rows_only(mx, fmt):
    x, w = acts(1, 70, 256), acts(2, 200, 256, torch.float32)
    x[3, 17], w[150, 255] = float("nan"), float("inf")
    t = 1.0 if fmt == "nvfp4" else None
    y = mx.linear(mx.quantize(x, fmt, tensor_scale=t), mx.quantize(w, fmt, tensor_scale=t))
    lost = torch.zeros_like(y, dtype=torch.bool)
    lost[3], lost[:, 150] = True, True
    assert torch.equal(torch.isnan(y), lost)


@pytest.mark.parametrize("fmt", FMTS)
def test_extreme_scales(mx, fmt):
    """Products of very small and very large blocks keep float32's range."""
    x, w = acts(1, 5, 128, torch.float32), acts(2, 130, 128, torch.float32)
    for a, b in ((2.0 ** 50, 2.0 ** 60), (2.0 ** -60, 2.0 ** -50), (2.0 ** -100, 2.0 ** 100)):
        q, p = mx.quantize(x * a, fmt), mx.quantize(w * b, fmt)
        xv, wv = q.dequantize().double(), p.dequantize().double()
        ref, mass = f64(xv @ wv.T), f64(xv.abs() @ wv.abs().T)
        assert_rounds(mx.linear(q, p), ref, sum_error(mass, 128))


def test_no_rows(mx):
    w = mx.quantize(torch.randn((8, 64), device="cuda"), "mxfp4")
    assert mx.linear(torch.empty((0, 64), device="cuda"), w).shape == (0, 8)
    q = mx.quantize(torch.empty((0, 64), device="cuda"), "nvfp4")
    assert q.dequantize().shape == (0, 64) and float(q.tensor_scale) == 1.0


GROUPS = [[1], [0, 0, 5], [3, 0, 64, 65, 0, 1], [0] * 20 + [1] + [0] * 43, [200, 1, 0, 130], [128, 256, 384],
          [700, 0, 90, 513], [2] * 100]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("sizes", GROUPS, ids=lambda s: f"{len(s)}groups{sum(s)}")
@pytest.mark.parametrize("N,K", [(96, 64), (300, 1000), (129, 2048)])
def test_linear_grouped(mx, fmt, sizes, N, K):
    E, R = len(sizes), sum(sizes)
    x = acts(R + N, R, K)
    w = (acts(K, E * N, K, torch.float32, 0.2) * 0.1).view(E, N, K)
    at = np.concatenate(([0], np.cumsum(sizes)))
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    t = (0.25, 2.0 ** -10) if fmt == "nvfp4" else (None, None)
    q, p = mx.quantize(x, fmt, tensor_scale=t[0], offsets=offsets), mx.quantize(w, fmt, tensor_scale=t[1])
    bias = torch.randn((E, N), device="cuda").to(torch.bfloat16)
    y, yb = mx.linear_grouped(q, p), mx.linear_grouped(q, p, bias=bias)
    xv, wv = q.dequantize().double(), p.dequantize().double()
    for e in range(E):
        a = xv[at[e]:at[e + 1]]
        ref, mass = f64(a @ wv[e].T), f64(a.abs() @ wv[e].abs().T)
        assert_rounds(y[at[e]:at[e + 1]], ref, sum_error(mass, K))
        want = ref + f64(bias[e])
        assert_rounds(yb[at[e]:at[e + 1]], want, sum_error(mass, K) + 2.0 ** -21 * np.abs(want))
    assert torch.equal(y, mx.linear_grouped(q, p))


def test_rows_of_no_group_are_left_alone(mx):
    x = acts(1, 40, 64)
    off = torch.tensor([4, 10, 30], dtype=torch.int32, device="cuda")
    q = mx.quantize(x, "mxfp4", offsets=off)
    w = mx.quantize(torch.randn((2, 48, 64), device="cuda"), "mxfp4")
    out = torch.full((40, 48), 7.0, device="cuda", dtype=torch.bfloat16)
    mx.linear_grouped(q, w, out=out)
    assert (out[:4] == 7).all() and (out[30:] == 7).all() and not (out[4:30] == 7).all(1).any()


def test_another_stream(mx):
    q, p, ref, mass = product_case(mx, "nvfp4", 48, 512, 1024)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = mx.linear(q, p)
    s.synchronize()
    assert_rounds(y, ref, sum_error(mass, 1024))


def test_products_in_a_graph(mx):
    x = acts(1, 4, 512)
    w = mx.quantize(acts(2, 384, 512, torch.float32), "mxfp4")
    mx.linear(x, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = mx.linear(x, w)
    x.copy_(acts(3, 4, 512))
    g.replay()
    assert torch.equal(y, mx.linear(x, w))


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(mx):
    from apsi_b200._lib import LowbitError
    x = torch.randn((4, 64), device="cuda")
    q, qn = mx.quantize(x, "mxfp4"), mx.quantize(x, "nvfp4")
    w3 = mx.quantize(torch.randn((2, 16, 64), device="cuda"), "mxfp4")
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    qg = mx.quantize(x, "mxfp4", offsets=off)
    bad = [
        lambda: mx.quantize(x, "mxfp8"), lambda: mx.quantize(x.cpu(), "mxfp4"), lambda: mx.quantize(x.double(), "mxfp4"),
        lambda: mx.quantize(x[0], "mxfp4"), lambda: mx.quantize(x.t(), "mxfp4"), lambda: mx.quantize(x.expand(4, 64)[:1].expand(4, 64), "mxfp4"),
        lambda: mx.quantize(x, "mxfp4", tensor_scale=1.0), lambda: mx.quantize(x, "nvfp4", tensor_scale=0.0),
        lambda: mx.quantize(x, "nvfp4", tensor_scale=torch.ones(2, device="cuda")),
        lambda: mx.quantize(x, "mxfp4", rows=torch.zeros(3, device="cuda", dtype=torch.int64)),
        lambda: mx.quantize(x, "mxfp4", offsets=off[:1]), lambda: mx.quantize(x[:, :0], "mxfp4"),
        lambda: mx.quantize(torch.randn((1025, 1, 32), device="cuda"), "mxfp4"),
        lambda: mx.dequantize(q, torch.float64), lambda: mx.plain_scales(qg),
        lambda: mx.pack(q.codes.int(), mx.plain_scales(q), 64, "mxfp4"), lambda: mx.pack(q.codes, mx.plain_scales(q)[:2], 64, "mxfp4"),
        lambda: mx.pack(q.codes, mx.plain_scales(q), 66, "mxfp4"),
        lambda: mx.linear(q, qn), lambda: mx.linear(qg, q), lambda: mx.linear(q, w3), lambda: mx.linear(q, x),
        lambda: mx.linear(mx.quantize(x[:, :32], "mxfp4"), q), lambda: mx.linear(q, q, accumulate=True),
        lambda: mx.linear(q, q, bias=torch.zeros(4, device="cuda")), lambda: mx.linear(q, q, out=torch.zeros((4, 4), device="cuda")),
        lambda: mx.linear(q, q, out=torch.zeros((4, 5), device="cuda", dtype=torch.bfloat16)),
        lambda: mx.linear(q, q, out=torch.zeros((4, 8), device="cuda", dtype=torch.bfloat16)[:, ::2]),
        lambda: mx.linear(q, q, out=torch.zeros((1, 4), device="cuda", dtype=torch.bfloat16).expand(4, 4)),
        lambda: mx.linear_grouped(q, w3), lambda: mx.linear_grouped(qg, q),
        lambda: mx.linear_grouped(qg, mx.quantize(torch.randn((3, 16, 64), device="cuda"), "mxfp4")),
        lambda: mx.linear_grouped(qg, w3, bias=torch.zeros(16, device="cuda", dtype=torch.bfloat16)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(LowbitError):
            f()
            pytest.fail(f"case {i} was taken")


def test_offsets_past_32_bits(mx):
    """More than 2^31 values: the last rows' codes, scales and values lie beyond 32-bit offsets."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    R, K = 40000, 57344
    x = torch.empty((R, K), device="cuda", dtype=torch.bfloat16)
    x[:8].normal_()
    x[8:-8] = 1.0
    x[-8:].normal_()
    q = mx.quantize(x, "mxfp4")
    ends = torch.cat((x[:8], x[-8:]))
    want = ora.quantize(f64(ends), "mxfp4")[2]
    v = q.dequantize(torch.bfloat16)
    assert np.array_equal(f64(torch.cat((v[:8], v[-8:]))), want)
    assert bool((v[8:-8] == 1).all())
    del v
    del x
    # the same codes as a weight of 40000 rows, read at both ends
    a = mx.quantize(torch.randn((3, K), device="cuda"), "mxfp4")
    y = mx.linear(a, q)
    ref = f64(a.dequantize().double()) @ want.T
    mass = np.abs(f64(a.dequantize().double())) @ np.abs(want).T
    assert_rounds(torch.cat((y[:, :8], y[:, -8:]), 1), ref, sum_error(mass, K))
