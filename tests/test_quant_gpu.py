"""GPU tests of the microscaled 4-bit operators (csrc/mxfp4.hip) against their definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def reference(x):
    """(codes [M, Kb, 32], scale bytes [M, Kb], values [M, K]) of x [M, K] in float64: nearest magnitude, halves to the even code."""
    a = x.detach().cpu().double().numpy()
    M, K = a.shape
    b = np.zeros((M, -(-K // 32) * 32))
    b[:, :K] = a
    b = b.reshape(M, -1, 32)
    fin = np.isfinite(b).all(-1)
    big = np.abs(np.where(fin[..., None], b, 0.0)).max(-1)
    e = np.where(big > 0, np.frexp(big)[1] - 1, -200) - 2
    e = np.maximum(e, -127)
    r = np.abs(np.where(fin[..., None], b, 0.0)) * np.exp2(-e)[..., None]
    code = np.zeros(r.shape, dtype=np.int64)
    for i in range(7):
        mid = (MAGNITUDES[i] + MAGNITUDES[i + 1]) / 2
        code += (r >= mid) if i % 2 else (r > mid)  # a half goes up from an odd code
    val = MAGNITUDES[code] * np.exp2(e)[..., None]
    sign = np.signbit(b)
    val = np.where(sign, -val, val)
    val[~fin] = np.nan
    return code + 8 * sign, np.where(fin, e + 127, 255), val.reshape(M, -1)[:, :K]


def unpack(q):
    """(codes [M, Kb', 32], scale bytes [M, Kb']) from the stored layout."""
    c = q.codes.cpu().numpy().transpose(1, 0, 2)  # [M, 8C, 16]
    codes = np.stack([c & 15, c >> 4], -1).reshape(q.M, -1, 32)
    s = q.scales.cpu().numpy().reshape(-1, 2, q.M, 4)  # [C, half, M, j]: block 8c + 2j + half
    return codes, s.transpose(2, 0, 3, 1).reshape(q.M, -1)


def check_quantised(x, q):
    code, sb, val = reference(x)
    got_c, got_s = unpack(q)
    nb = sb.shape[1]
    assert np.array_equal(got_s[:, :nb], sb)
    fin = sb != 255
    assert np.array_equal(got_c[:, :nb][fin], code[fin])
    assert (got_c[:, nb:] == 0).all()  # the padding
    dec = q.float().cpu().double().numpy().reshape(q.M, q.K)
    assert np.array_equal(dec, val, equal_nan=True)
    assert np.array_equal(np.signbit(dec)[~np.isnan(val)], np.signbit(val)[~np.isnan(val)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 32), (33, 31), (64, 256), (31, 257), (3, 1003), (100, 1280), (65, 4100)])
def test_quantize_vs_reference(M, K, dtype):
    from samnerf_amd import ops
    g = torch.Generator().manual_seed(M * 7919 + K)
    x = (torch.randn((M, K), generator=g) * torch.exp(3 * torch.randn((M, 1), generator=g))).to(dtype)
    q = ops.quantize_mxfp4(x.cuda())
    assert (q.M, q.K, q.shape) == (M, K, (M, K))
    check_quantised(x, q)
    back = ops.dequantize_mxfp4(q, dtype)  # exact in the type that was quantised
    assert back.dtype == dtype and torch.equal(back.float(), q.float())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,extra", [(0, 8), (0, 3), (1, 0), (5, 11)])
def test_quantize_strided_rows(offset, extra, dtype):
    """Rows of a wider matrix, from an address and with a stride that 16 bytes do not divide; NaN around them is not read."""
    from samnerf_amd import ops
    M, K = 37, 200
    g = torch.Generator().manual_seed(offset + extra)
    buf = torch.full((offset + M * (K + extra),), float("nan"), dtype=dtype, device="cuda")
    x = torch.as_strided(buf, (M, K), (K + extra, 1), offset)
    x.copy_(torch.randn((M, K), generator=g).to(dtype))
    check_quantised(x, ops.quantize_mxfp4(x))
    check_quantised(x.t().contiguous(), ops.quantize_mxfp4(x.t()))  # columns as rows: copied


def test_quantize_rounding_saturation_and_extremes():
    from samnerf_amd import ops
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0, 7.99, 6.0, 4.0]
    rows = []
    for s in (-127, -126, -60, 0, 60, 125):
        for base in (4.0, 7.9):  # the block's scale is s for both
            v = [base] + mids + [-m for m in mids] + [0.0, -0.0, 1e-3, -1e-3, 0.2499999, 0.2500001, 5.0000005]
            rows.append([math.ldexp(a, s) for a in v[:32]] + [0.0] * (32 - len(v[:32])))
    rows.append([0.0] * 32)
    rows.append([2.0 ** -149] + [0.0] * 31)
    rows.append([-(2.0 ** -127), 2.0 ** -128] + [0.0] * 30)
    x = torch.tensor(rows, dtype=torch.float64).float()
    check_quantised(x, ops.quantize_mxfp4(x.cuda()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_non_finite_blocks(dtype):
    """A block with an inf or a NaN reads back as NaN; its neighbours in the row are as ever."""
    from samnerf_amd import ops
    x = torch.randn((6, 96), generator=torch.Generator().manual_seed(0)).to(dtype)
    x[0, 40], x[1, 64], x[2, 0] = float("inf"), float("nan"), float("-inf")
    q = ops.quantize_mxfp4(x.cuda())
    check_quantised(x, q)
    w = ops.quantize_mxfp4(torch.randn((5, 96), generator=torch.Generator().manual_seed(1)).cuda())
    for M in (6, 70):  # through the product: exactly these rows
        y = ops.linear_mxfp4(torch.cat([x.cuda()] + [x[3:4].cuda()] * (M - 6)), w)
        assert torch.isnan(y[:3]).all() and torch.isfinite(y[3:]).all()


def test_quantize_shapes_and_empty():
    from samnerf_amd import ops
    x = torch.randn((2, 3, 40), generator=torch.Generator().manual_seed(0))
    q = ops.quantize_mxfp4(x.cuda())
    assert q.shape == (2, 3, 40) and q.M == 6 and q.float().shape == (2, 3, 40)
    check_quantised(x.view(6, 40), q)
    e = ops.quantize_mxfp4(torch.empty((0, 40), device="cuda"))
    assert e.M == 0 and e.float().shape == (0, 40)
    w = ops.quantize_mxfp4(torch.randn((7, 40), device="cuda"))
    assert ops.linear_mxfp4(torch.empty((0, 40), device="cuda"), w).shape == (0, 7)
    v = ops.quantize_mxfp4(x[0, 0].cuda())
    assert v.shape == (40,) and ops.linear_mxfp4(x[0, 0].cuda(), w).shape == (7,)


def test_quantize_writes_nothing_else():
    from samnerf_amd import ops
    from samnerf_amd import _opcore as C
    M, K = 37, 300
    x = torch.randn((M, K), device="cuda")
    codes = torch.full((16 * M * 16 + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((4 * M * 4 + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.full((M * K + 1024,), 7.0, device="cuda")
    C._launch("snf_mxfp4_quantize", C._p(x), 0, M, K, K, C._p(codes), C._p(scales), C._stream())
    C._launch("snf_mxfp4_dequantize", C._p(codes), C._p(scales), M, K, C._p(out), 0, C._stream())
    assert (codes[16 * M * 16:] == 0xA5).all() and (scales[4 * M * 4:] == 0xA5).all() and (out[M * K:] == 7.0).all()
    w = ops.quantize_mxfp4(torch.randn((21, K), device="cuda"))
    q = ops.quantize_mxfp4(x)
    y = torch.full((M * 21 + 1024,), 7.0, device="cuda")
    C._launch("snf_mxfp4_linear", C._p(q.codes), C._p(q.scales), C._p(w.codes), C._p(w.scales), None, M, K, 21, 0, C._p(y), 0, C._stream())
    assert (y[M * 21:] == 7.0).all()


def test_quantize_offsets_past_32_bits():
    """More than 2^32 bytes of codes and 2^33 values: the last rows come back as the first."""
    from samnerf_amd import ops
    base = torch.randn((1024, 8192), device="cuda", dtype=torch.bfloat16)
    x = base.repeat(1030, 1)
    q = ops.quantize_mxfp4(x)
    assert q.codes.numel() > 1 << 32
    del x
    y = ops.dequantize_mxfp4(q, torch.bfloat16)
    want = ops.dequantize_mxfp4(ops.quantize_mxfp4(base), torch.bfloat16)
    assert torch.equal(y[:1024], want) and torch.equal(y[-1024:], want)
    w = ops.quantize_mxfp4(torch.randn((8, 8192), device="cuda"))
    z = ops.linear_mxfp4(q, w)
    one = ops.linear_mxfp4(ops.Mxfp4(q.codes[:, :4096].contiguous(), q.scales[:, :4096].contiguous(), 8192), w)
    assert torch.equal(z[:4096], one) and torch.equal(z[-1024:], one[:1024])


# ---- product ------------------------------------------------------------------------------------------------------------------------
def act64(y, act):
    return {0: lambda v: v, 1: lambda v: torch.where(v > 0, v, torch.zeros_like(v)), 2: torch.sigmoid,
            3: lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2.0))}[act](y)


def product_error(y, xv, wv, bias, act):
    """Largest |y - exact| over its bound.  Sums: products of codes are exact, K additions of at most half a step of the running sum
    each, K 2^-24 sum|a w| (and the bias' addition).  The activations' slopes are at most 1.13; exp / erf and the operations around
    them add 8 steps of at most max(|y|, |value|).  The last rounding: half a step of the type (or half its smallest subnormal)."""
    s = xv @ wv.t()
    mag = xv.abs() @ wv.abs().t()
    if bias is not None:
        s = s + bias
        mag = mag + bias.abs()
    K = xv.shape[1]
    exact = act64(s, act)
    tol = (K + 1) * 2.0 ** -24 * mag * 1.13
    if act in (2, 3):
        tol = tol + 8 * 2.0 ** -24 * torch.maximum(exact.abs(), s.abs() if act == 3 else torch.ones_like(s))
    fi = torch.finfo(y.dtype)
    tol = tol * (1 + fi.eps) + exact.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps
    return float(((y.cpu().double() - exact).abs() / tol.clamp_min(1e-300)).max())


SIZES = [(1, 1, 1), (1, 37, 1280), (2, 64, 33), (7, 130, 100), (16, 100, 515), (17, 33, 300), (40, 48, 64), (64, 777, 1003), (65, 1, 700),
         (333, 777, 1003), (129, 127, 257), (300, 5, 96), (300, 16, 2000), (128, 256, 512), (520, 260, 1300), (1030, 17, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear_vs_reference(M, N, K, dtype):
    from samnerf_amd import ops
    g = torch.Generator().manual_seed(M + 3 * N + 7 * K)
    x = (torch.randn((M, K), generator=g) * torch.exp(torch.randn((1, K), generator=g))).to(dtype)
    w = torch.randn((N, K), generator=g) / math.sqrt(K)
    bias = torch.randn((N,), generator=g)
    wq = ops.quantize_mxfp4(w.cuda())
    xv, wv = torch.from_numpy(reference(x)[2]), torch.from_numpy(reference(w)[2])
    for act, b in ((0, None), (3, bias), (1, bias), (2, None)):
        y = ops.linear_mxfp4(x.cuda(), wq, None if b is None else b.cuda(), act=act)
        assert y.dtype == dtype and y.shape == (M, N)
        assert product_error(y, xv, wv, None if b is None else b.double(), act) <= 1.0
    q = ops.quantize_mxfp4(x.cuda())
    for od in DTYPES:  # an operand quantised before, every result type
        y = ops.linear_mxfp4(q, wq, bias.cuda(), out_dtype=od)
        assert y.dtype == od and product_error(y, xv, wv, bias.double(), 0) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,act", [(8200, 8180, 300, 3), (8192, 8192, 64, 0), (8449, 7937, 257, 1), (1025, 1100, 700, 3), (2000, 1031, 96, 2)])
def test_linear_tiles_vs_reference(M, N, K, act, dtype):
    """Sizes that the two tile kernels take, whole tiles and ragged ones: against the decoded operands' product in 64 bits."""
    from samnerf_amd import ops
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    x = torch.randn((M, K), generator=g, device="cuda").to(dtype)
    wq = ops.quantize_mxfp4(torch.randn((N, K), generator=g, device="cuda") / math.sqrt(K))
    bias = torch.randn((N,), generator=g, device="cuda")
    xq = ops.quantize_mxfp4(x)
    y = ops.linear_mxfp4(x, wq, bias, act=act)
    xv, wt = xq.float().double(), wq.float().double().t().contiguous()
    s = xv @ wt + bias.double()
    mag = xv.abs() @ wt.abs() + bias.double().abs()
    exact = act64(s, act)
    tol = (K + 1) * 2.0 ** -24 * mag * 1.13  # (as product_error)
    if act in (2, 3):
        tol += 8 * 2.0 ** -24 * torch.maximum(exact.abs(), s.abs() if act == 3 else torch.ones_like(s))
    fi = torch.finfo(dtype)
    tol = tol * (1 + fi.eps) + exact.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps
    assert bool(((y.double() - exact).abs() <= tol).all())


@pytest.mark.parametrize("M,N,K", [(1, 640, 320), (50, 70, 320), (200, 130, 4100)])
def test_linear_scales_far_apart(M, N, K):
    """Blocks whose scales differ by up to 2^40 on both sides, and rows of zeros."""
    from samnerf_amd import ops
    g = torch.Generator().manual_seed(K)
    x = torch.randn((M, K), generator=g) * torch.exp2(torch.randint(-20, 20, (M, K), generator=g).float())
    w = torch.randn((N, K), generator=g) * torch.exp2(torch.randint(-20, 20, (N, K), generator=g).float())
    x[M // 2], w[N // 3] = 0.0, 0.0
    y = ops.linear_mxfp4(x.cuda(), ops.quantize_mxfp4(w.cuda()))
    assert product_error(y, torch.from_numpy(reference(x)[2]), torch.from_numpy(reference(w)[2]), None, 0) <= 1.0
    assert (y[:, N // 3] == 0).all() and (y[M // 2] == 0).all()


@pytest.mark.parametrize("M", [1, 5, 40, 300])
def test_linear_strided_input_and_views(M):
    from samnerf_amd import ops
    K, N = 200, 90
    buf = torch.full((M * 211 + 3,), float("nan"), device="cuda")
    x = torch.as_strided(buf, (M, K), (211, 1), 3)
    x.copy_(torch.randn((M, K), device="cuda"))
    w = ops.quantize_mxfp4(torch.randn((N, K), device="cuda"))
    want = ops.linear_mxfp4(x.contiguous(), w)
    assert torch.equal(ops.linear_mxfp4(x, w), want)
    assert torch.equal(ops.linear_mxfp4(x.contiguous().view(M, 1, K), w).view(M, N), want)
    big = torch.randn((4 * N,), device="cuda")  # a bias at an odd address, and one with a stride
    assert torch.equal(ops.linear_mxfp4(x, w, big[1:N + 1]), ops.linear_mxfp4(x, w, big[1:N + 1].clone()))
    assert torch.equal(ops.linear_mxfp4(x, w, big[::4]), ops.linear_mxfp4(x, w, big[::4].clone()))


@pytest.mark.parametrize("M,N", [(1, 300), (30, 300), (1100, 1111), (8200, 8180)])
def test_linear_repeats_streams_and_graphs(M, N):
    """The same bits again, on another stream, and from a replayed graph with new inputs."""
    from samnerf_amd import ops
    K = 1300 if M < 8000 else 300
    w = ops.quantize_mxfp4(torch.randn((N, K), device="cuda"))
    xs = [torch.randn((M, K), device="cuda") for _ in range(3)]
    want = [ops.linear_mxfp4(x, w, act=ops.ACT_GELU) for x in xs]
    assert torch.equal(ops.linear_mxfp4(xs[0], w, act=ops.ACT_GELU), want[0])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = ops.linear_mxfp4(xs[1], w, act=ops.ACT_GELU)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(y, want[1])
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear_mxfp4(x, w, act=ops.ACT_GELU)
    for i in (1, 2, 0):
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(ops.linear_mxfp4(xs[i], w, act=ops.ACT_GELU), want[i])  # eager work in between
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])


def test_refusals_on_the_device():
    from samnerf_amd import _lib, ops
    from samnerf_amd import _opcore as C
    w = ops.quantize_mxfp4(torch.randn((8, 64), device="cuda"))
    x = torch.randn((3, 64), device="cuda")
    with pytest.raises(RuntimeError):
        ops.linear_mxfp4(x.cpu(), w)
    with pytest.raises(ValueError):
        ops.linear_mxfp4(x[:, :63], w)
    with pytest.raises(ValueError):
        ops.linear_mxfp4(x, w, torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError):
        ops.linear_mxfp4(x, w, torch.zeros(8, device="cuda", dtype=torch.float16))
    with pytest.raises(RuntimeError):
        ops.linear_mxfp4(x, w, torch.zeros(8))
    with pytest.raises(ValueError):
        ops.linear_mxfp4(x, w, act=4)
    for args in ((C._p(x), 7, 3, 64, 64), (C._p(x), 0, 3, 0, 64), (C._p(x), 0, -1, 64, 64), (C._p(x), 0, 3, 64, 63), (None, 0, 3, 64, 64)):
        with pytest.raises(_lib.SnfError):
            C._launch("snf_mxfp4_quantize", *args, C._p(w.codes), C._p(w.scales), C._stream())
    with pytest.raises(_lib.SnfError):
        C._launch("snf_mxfp4_linear", C._p(w.codes) + 4, C._p(w.scales), C._p(w.codes), C._p(w.scales), None, 3, 64, 8, 0, C._p(x), 0, C._stream())
    with pytest.raises(_lib.SnfError):
        C._launch("snf_mxfp4_linear", C._p(w.codes), C._p(w.scales), C._p(w.codes), C._p(w.scales), None, 3, 64, 8, 9, C._p(x), 0, C._stream())


@pytest.mark.parametrize("M,K", [(1, 8), (70, 40), (64, 256), (130, 264), (33, 1280)])
def test_quantize_planes_vs_rows(M, K):
    """The encoder's operand planes hold hi + lo: the codes of that sum."""
    from samnerf_amd import ops
    x = torch.randn((M, K), generator=torch.Generator().manual_seed(K)) * 3
    planes = ops.split_planes_kb(x.cuda())
    q = ops.quantize_mxfp4(planes)
    check_quantised(planes.float().cpu(), q)
    w = ops.quantize_mxfp4(torch.randn((9, K), device="cuda"))
    assert torch.equal(ops.linear_mxfp4(planes, w), ops.linear_mxfp4(q, w))


@pytest.mark.parametrize("M,N,K", [(1, 256, 32), (5, 40, 64), (37, 512, 100), (130, 256, 1003), (300, 1280, 320), (700, 100, 256), (8200, 8192, 64)])
def test_linear_quantized_result(M, N, K):
    """The next layer's operand from the product itself: the codes of its float32 result (the two kernels may add in another order where
    one deals k out among waves: those sizes are compared by value, to a step of a block's scale)."""
    from samnerf_amd import ops
    g = torch.Generator().manual_seed(M + N + K)
    x, w, b = torch.randn((M, K), generator=g).cuda(), torch.randn((N, K), generator=g).cuda(), torch.randn((N,), generator=g).cuda()
    wq = ops.quantize_mxfp4(w)
    xq = ops.quantize_mxfp4(x)
    for act in (0, 3):
        q = ops.linear_mxfp4(x.view(M, 1, K), wq, b, act=act, quantized=True)
        assert isinstance(q, ops.Mxfp4) and q.shape == (M, 1, N)
        y = ops.linear_mxfp4(xq, wq, b, act=act)
        want = ops.quantize_mxfp4(y)
        if -(-M // 128) * -(-N // 128) >= 64 or N % 256:
            assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)
        else:  # one rounding border crossed moves a value by a code, 2 scales at most; a scale that doubles rounds to twice the step.  The two
            # sums differ by at most 2 K 2^-24 sum|a w|, under 1e-3 of a block's smallest step (scale / 2): less than 1 % lie that near to one
            step = y.view(M, -1).abs().amax(dim=1, keepdim=True) / 2
            assert bool(((q.float().view(M, N) - want.float()).abs() <= step).all())
            assert float((q.float().view(M, N) != want.float()).float().mean()) <= 0.01
    e = ops.linear_mxfp4(x[:0], wq, b, quantized=True)
    assert e.M == 0 and e.shape == (0, N)
    with pytest.raises(ValueError):
        ops.linear_mxfp4(x, wq, b, out_dtype=torch.float16, quantized=True)


def test_gelu_far_out_and_not_finite():
    """The activation at both ends: 0 and the value itself; an infinite sum gives its limit, a NaN stays one."""
    from samnerf_amd import ops
    w = ops.quantize_mxfp4(torch.ones((1, 32), device="cuda"))
    x = torch.zeros((9, 32), device="cuda")
    v = torch.tensor([-40.0, -9.0, -1e-3, 0.0, 1e-3, 9.0, 40.0, 0.0, 0.0], device="cuda")
    x[:, 0] = 0.0
    for M in (9, 40, 8200):  # every kernel of the product
        xs = x.repeat(-(-M // 9), 1)[:M]
        for i, b in enumerate(v.tolist()[:7]):
            y = ops.linear_mxfp4(xs, w, torch.full((1,), b, device="cuda"), act=ops.ACT_GELU)
            want = 0.5 * b * math.erfc(-b / math.sqrt(2.0))
            assert float((y.double() - want).abs().max()) <= 8 * 2.0 ** -24 * abs(b)
        for b, want in ((math.inf, math.inf), (-math.inf, 0.0), (math.nan, math.nan)):
            y = ops.linear_mxfp4(xs, w, torch.full((1,), b, device="cuda"), act=ops.ACT_GELU)
            assert bool((torch.isnan(y) if math.isnan(want) else y == want).all())


# ---- the encoder in this format -------------------------------------------------------------------------------------------------------
def _small_encoder(embed, depth=2, window=5):
    from functools import partial
    from samnerf_amd.image_encoder import ImageEncoderViT
    torch.manual_seed(embed)
    enc = ImageEncoderViT(img_size=224, patch_size=16, embed_dim=embed, depth=depth, num_heads=4, mlp_ratio=2.0, out_chans=32, qkv_bias=True,
                          norm_layer=partial(torch.nn.LayerNorm, eps=1e-6), use_rel_pos=True, window_size=window,
                          global_attn_indexes=(depth - 1,))
    with torch.no_grad():
        for p in enc.parameters():
            if p.dim() > 1:
                p.normal_(0, 0.05)
    return enc.cuda().eval()


@pytest.mark.parametrize("embed", [64, 256])  # the plain path and the one on operand planes
def test_encoder_blocks_compute_what_their_layers_say(embed, monkeypatch):
    """Every dense layer of every block goes through the product once, in order, with its own quantised weight and bias, and each result
    is the exact product of its operands to the bound of product_error; the other format is as before afterwards."""
    from samnerf_amd import ops
    enc = _small_encoder(embed)
    x = torch.randn((1, 3, 224, 224), generator=torch.Generator().manual_seed(1)).cuda()
    split = enc(x)
    enc.set_linear_format("mxfp4")
    y = enc(x)
    layers = [l for blk in enc.blocks for l in (blk.attn.qkv, blk.attn.proj, blk.mlp.lin1, blk.mlp.lin2)]
    real, seen = ops.linear_mxfp4, []

    def checked(a, w, bias=None, act=0, **kw):
        r = real(a, w, bias, act, **kw)
        lin = layers[len(seen)]
        seen.append(lin)
        assert bias is lin.bias and torch.equal(w.float(), ops.quantize_mxfp4(lin.weight.detach()).float())
        q = a if isinstance(a, ops.Mxfp4) else ops.quantize_mxfp4(a)
        values = r.float() if isinstance(r, ops.Mxfp4) else r
        if not isinstance(r, ops.Mxfp4):
            assert product_error(values.reshape(-1, w.M), q.float().view(-1, w.K).cpu().double(), w.float().cpu().double(),
                                 bias.detach().cpu().double(), act) <= 1.0
        return r

    monkeypatch.setattr(ops, "linear_mxfp4", checked)
    z = enc(x)
    monkeypatch.undo()
    assert seen == layers and torch.equal(y, z)
    assert y.shape == split.shape and bool(torch.isfinite(y).all()) and not torch.equal(y, split)
    enc.set_linear_format("split")
    assert torch.equal(enc(x), split)


def test_encoder_weights_are_requantised_when_written():
    enc = _small_encoder(64).set_linear_format("mxfp4")
    x = torch.randn((1, 3, 224, 224), generator=torch.Generator().manual_seed(1)).cuda()
    a = enc(x)
    with torch.no_grad():
        enc.blocks[0].attn.qkv.weight.mul_(0.5)
    b = enc(x)
    assert not torch.equal(a, b)
    with torch.no_grad():
        enc.blocks[0].attn.qkv.weight.mul_(2.0)
    assert torch.equal(enc(x), a)
    with pytest.raises(ValueError):
        enc.set_linear_format("fp4")


@pytest.mark.parametrize("fmt", ["split", "mxfp4"])
def test_encoder_on_two_streams(fmt):
    """A first forward on a busy stream and one on another right behind it, and forwards of both streams at once: each as alone (weights
    that a cache holds are whole, operand planes are a stream's own)."""
    enc = _small_encoder(256).set_linear_format(fmt)
    g = torch.Generator().manual_seed(1)
    xs = [torch.randn((1, 3, 224, 224), generator=g).cuda() for _ in range(4)]
    want = [enc(x) for x in xs]
    enc.reset_weight_cache()
    side = torch.cuda.Stream()
    a = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            a = (a @ a).clamp_(-1.0, 1.0)
        first = enc(xs[0])
    second = enc(xs[1])
    torch.cuda.synchronize()
    assert torch.equal(first, want[0]) and torch.equal(second, want[1])
    got = []
    for i in range(12):
        with torch.cuda.stream(side):
            got.append((2 * (i % 2), enc(xs[2 * (i % 2)])))
        got.append((2 * (i % 2) + 1, enc(xs[2 * (i % 2) + 1])))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)


@pytest.mark.parametrize("cold", [True, False])
@pytest.mark.parametrize("fmt", ["split", "mxfp4"])
@pytest.mark.parametrize("embed", [64, 256])
def test_encoder_captured(embed, fmt, cold):
    """A captured forward replays as the eager one, with eager forwards in between; one captured before anything was cached leaves nothing in
    the cache that only its replays write; one that read the cache keeps what it read, also after the weights were written."""
    enc = _small_encoder(embed).set_linear_format(fmt)
    g = torch.Generator().manual_seed(2)
    xs = [torch.randn((1, 3, 224, 224), generator=g).cuda() for _ in range(3)]
    want = [enc(x) for x in xs]
    if cold:
        enc.reset_weight_cache()
        enc._pcache.clear()
    torch.cuda.synchronize()
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = enc(x)
    assert torch.equal(enc(xs[1]), want[1])  # before any replay
    for i in (2, 0, 1):
        x.copy_(xs[i])
        graph.replay()
        eager = enc(xs[(i + 1) % 3])
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and torch.equal(eager, want[(i + 1) % 3])
    cached = fmt == "mxfp4" or embed == 256  # (the plain path of the other format reads the parameters themselves)
    with torch.no_grad():
        enc.blocks[0].attn.qkv.weight.mul_(0.5)
    new = enc(xs[1])
    junk = [torch.full((1 << 22,), float("nan"), device="cuda") for _ in range(8)]  # (what was freed is written again)
    graph.replay()
    torch.cuda.synchronize()
    del junk
    assert not torch.equal(new, want[1])
    assert torch.equal(y, want[1] if cached and not cold else new)


def test_encoder_weights_that_are_replaced():
    """A new parameter in a layer is a new weight, also where it lies at the address of an earlier one that is gone."""
    from samnerf_amd import ops
    enc = _small_encoder(64)
    lin = enc.blocks[0].attn.qkv
    shape = lin.weight.shape
    for i in range(40):
        lin.weight = None
        lin.weight = torch.nn.Parameter(torch.full(shape, float(i + 1), device="cuda"))
        assert torch.equal(enc._wmxfp4(lin).float(), ops.quantize_mxfp4(lin.weight.detach()).float())
        hi, lo = enc._wplanes(lin)
        assert bool((hi.float() + lo.float() == i + 1).all())


@pytest.mark.parametrize("embed", [64, 256])  # the plain path and the one on operand planes
def test_encoder_layers_are_fed_and_used_as_the_block_says(embed, monkeypatch):
    """The blocks' formulas in 64 bits around the layers' own results: the encoder in 4 bits hands every dense layer the operand that the
    formulas make of the results before it (norms, windows, attention, residuals: 2^-16 of a product's operands, scores up to 10, so 2e-3
    of the largest value), lin1 alone applies the GELU, and its result is the quantised product of its operands; what comes out is what the
    formulas make of the last results."""
    from samnerf_amd import ops
    from oracle import vit_oracle as V
    enc = _small_encoder(embed).set_linear_format("mxfp4")
    x = torch.randn((2, 3, 224, 224), generator=torch.Generator().manual_seed(3)).cuda()
    real, calls = ops.linear_mxfp4, []

    def recorded(a, w, bias=None, act=0, **kw):
        r = real(a, w, bias, act, **kw)
        rows = lambda t: t.float().cpu().double().clone()  # noqa: E731  (operand planes are written again by the next block)
        calls.append((rows(a), rows(w), None if bias is None else rows(bias.detach()), act, isinstance(a, ops.Mxfp4), isinstance(r, ops.Mxfp4), rows(r)))
        return r

    monkeypatch.setattr(ops, "linear_mxfp4", recorded)
    y, trace = enc(x, trace_blocks=(0, 1))
    names = ["qkv", "proj", "lin1", "lin2"] * 2
    assert len(calls) == 8 and [c[3] for c in calls] == [ops.ACT_GELU if n == "lin1" else ops.ACT_NONE for n in names]
    # lin1: the codes of its float32 result (a sum next to a border may fall on the other side: test_linear_quantized_result)
    for (a, w, b, act, _, codes, r), n in zip(calls, names):
        assert codes == (n == "lin1")
        if codes:
            values = lambda t: torch.from_numpy(reference(t)[2])  # noqa: E731
            want = values(act64(values(a) @ w.t() + b, 3).float())
            assert bool(((r - want).abs() <= want.abs().amax(1, keepdim=True) / 2).all()) and float((r != want).double().mean()) <= 0.01
            dropped = values((values(a) @ w.t() + b).float())
            assert float((r != dropped).double().mean()) > 0.3  # (the comparison sees a missing GELU)
    left = list(zip(calls, names))

    class Formulas:
        layer_norm, pad, conv2d = torch.nn.functional.layer_norm, torch.nn.functional.pad, torch.nn.functional.conv2d
        gelu = staticmethod(lambda t: t)  # (lin1's results are after it)

        @staticmethod
        def linear(t, w, b):
            (a, wv, bv, _, coded, _, r), n = left.pop(0)
            got = a.reshape(-1, w.shape[1])
            rows = t.reshape(-1, w.shape[1])
            assert got.shape == rows.shape and float((got - rows).abs().max()) <= (0 if coded else 2e-3 * float(rows.abs().max())), n
            assert coded == (n == "lin2")
            assert torch.equal(wv, torch.from_numpy(reference(w)[2])) and torch.equal(bv, b)
            return r.reshape(*t.shape[:-1], w.shape[0])

    monkeypatch.setattr(V, "F", Formulas)
    cfg = V.ViTConfig(img_size=224, patch_size=16, embed_dim=embed, depth=2, num_heads=4, mlp_ratio=2.0, out_chans=32, window_size=5,
                      global_attn_indexes=(1,))
    sd = {k: v.detach().cpu().double() for k, v in enc.state_dict().items()}
    want, tokens = V.forward(sd, x.cpu().double(), cfg, return_tokens=True)
    assert not left
    for i in (0, 1):
        assert float((trace[i].cpu().double() - tokens[i + 1]).abs().max()) <= 2e-3 * float(tokens[i + 1].abs().max())
    assert float((y.cpu().double() - want).abs().max()) <= 2e-3 * float(want.abs().max())
