"""GPU tests of a teacher's top logits and the distillation loss that reads them (csrc/distill.hip), against their definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of float32, relative


# ---- top logits ---------------------------------------------------------------------------------------------------------------------
def top64(x, k, T):
    """(ids, logits, rest) in float64 on the CPU; NaN above everything, equal logits in the order of their places."""
    x = x.detach().cpu().double()
    v, order = torch.sort(x, dim=1, descending=True, stable=True)
    others = v[:, k:]
    rest = torch.logsumexp(others / T, dim=1) if others.shape[1] else torch.full((x.shape[0],), -math.inf, dtype=torch.float64)
    return order[:, :k].to(torch.int32), v[:, :k], rest


def check_top(x, k, T, got):
    ids, v, rest = top64(x, k, T)
    assert torch.equal(got.ids.cpu(), ids)
    assert torch.equal(torch.nan_to_num(got.logits.cpu().double(), nan=12345.0), torch.nan_to_num(v, nan=12345.0))
    # m / T + log sum: the sum's terms carry |x - m| / T 2^-24 for their exponents (at most 88 before they vanish) and a few steps of exp,
    # weighted by their share: under 20 steps together; its n additions run over at most 128 terms a thread and a tree of 9 levels
    r = got.rest.cpu().double()
    tol = U * (200 + 4 * (rest.abs() + (v[:, -1].abs() / T)).nan_to_num(0.0, 0.0, 0.0))
    same = (r == rest) | (torch.isnan(r) & torch.isnan(rest))
    assert bool((same | ((r - rest).abs() <= tol)).all())


TOP_SIZES = [(1, 1, 1), (3, 2, 2), (5, 17, 17), (4, 64, 5), (7, 100, 64), (2, 257, 256), (33, 192, 8), (5, 1003, 16), (3, 1003, 64),
             (1, 2047, 3), (2, 4100, 200), (300, 4096, 32), (1, 32000, 8), (260, 20011, 48), (2, 65536, 64), (1, 100003, 256), (1, 400000, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,k", TOP_SIZES)
def test_top_logits_vs_reference(R, V, k, dtype):
    from samnerf_amd import ops
    g = torch.Generator().manual_seed(R + V + k)
    x = (3 * torch.randn((R, V), generator=g)).to(dtype)
    for T in (1.0, 2.5):
        check_top(x, k, T, ops.top_logits(x.cuda(), k, temperature=T))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(40, 7), (1003, 40), (5000, 64), (70001, 130)])
def test_top_logits_ties_and_runs(V, k, dtype):
    """Rows of few different values, constant rows, ascending and descending rows, -0 beside 0."""
    from samnerf_amd import ops
    g = torch.Generator().manual_seed(V)
    rows = [torch.randint(0, 3, (V,), generator=g).float(), torch.zeros(V), torch.full((V,), -2.5), torch.arange(V) / V, -torch.arange(V) / V,
            torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0), torch.where(torch.arange(V) < V - 3, 0.0, 5.0)]
    x = torch.stack(rows).to(dtype)
    check_top(x, k, 1.5, ops.top_logits(x.cuda(), k, temperature=1.5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(40, 7), (3000, 64), (70001, 130)])
def test_top_logits_infinities_nan_and_masks(V, k, dtype):
    from samnerf_amd import ops
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(V)
    x = torch.randn((9, V), generator=g)
    x[0] = -math.inf                       # nothing left
    x[1, 3:] = -math.inf                   # fewer finite logits than k
    x[2] = low                             # the type's lowest value everywhere
    x[3, k // 2:] = low
    x[4, V // 2] = math.nan
    x[5, ::3] = math.nan                   # more NaN than k
    x[6, 5] = math.inf
    x[7, ::2] = math.inf                   # more infinities than k
    x[8, :k] += 1000.0 if dtype != torch.float16 else 600.0   # the rest far below
    x = x.to(dtype)
    check_top(x, k, 1.0, ops.top_logits(x.cuda(), k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(60, 7), (3000, 40), (70001, 130), (300000, 256)])
def test_top_logits_runs_with_gaps(V, k, dtype):
    """Runs of equal logits around the k-th, between far lower ones and a NaN: nothing of the top reaches the rest's reference."""
    from samnerf_amd import ops
    g = torch.Generator().manual_seed(V)
    high = 600.0 if dtype == torch.float16 else 2000.0
    x = torch.randn((7, V), generator=g)
    x[0, V // 3:V // 3 + k] = high                       # exactly k equals, the rest far below
    x[1, V // 3:V // 3 + k - 1] = high                   # ... beside a NaN: k together
    x[1, 2] = math.nan
    x[2, V // 2:] = high                                 # one run that is longer than k, at the end
    x[3, torch.randperm(V, generator=g)[:V // 2]] = high  # scattered equals
    x[3, V - 1] = 2 * high
    x[4] = torch.sort(x[4]).values                       # ascending: the last groups
    x[5, :V // 2] = -math.inf                            # only a run behind masked places
    x[5, V // 2:] = -high
    x[6] = torch.relu(x[6] - 2.0)                        # few different values, most equal
    x = x.to(dtype)
    check_top(x, k, 1.0, ops.top_logits(x.cuda(), k))
    buf = torch.full((7, V + 5), math.inf, dtype=dtype, device="cuda")
    buf[:, 3:V + 3] = x.cuda()
    check_top(x, k, 1.0, ops.top_logits(buf[:, 3:V + 3], k))


@pytest.mark.parametrize("dtype", DTYPES)
def test_top_logits_rows_at_any_address(dtype):
    """Strided rows that start anywhere in a 16-byte granule; what lies between them is never taken."""
    from samnerf_amd import ops
    for off, V, extra, k in ((1, 333, 6, 9), (3, 1000, 1, 30), (0, 50, 7, 50), (5, 20000, 3, 8)):
        buf = torch.full((off + 6 * (V + extra) + 9,), math.inf, dtype=dtype, device="cuda")
        x = torch.as_strided(buf, (6, V), (V + extra, 1), off)
        x.copy_(torch.randn((6, V), generator=torch.Generator().manual_seed(V)).to(dtype))
        check_top(x, k, 1.0, ops.top_logits(x, k))
        assert torch.equal(ops.top_logits(x.t().contiguous().t(), k).ids, ops.top_logits(x, k).ids)


def test_top_logits_shapes():
    from samnerf_amd import ops
    x = torch.randn((2, 3, 50), device="cuda")
    t = ops.top_logits(x, 4)
    f = ops.top_logits(x.view(6, 50), 4)
    assert t.ids.shape == (2, 3, 4) and t.rest.shape == (2, 3)
    assert torch.equal(t.ids.view(6, 4), f.ids) and torch.equal(t.rest.view(6), f.rest)
    v = ops.top_logits(x[1, 2], 4)
    assert v.ids.shape == (4,) and v.rest.shape == () and torch.equal(v.ids, f.ids[5])
    e = ops.top_logits(x[:0], 4)
    assert e.ids.shape == (0, 3, 4) and e.rest.shape == (0, 3)


def test_top_logits_offsets_past_32_bits():
    """5 GB of logits, more than 2^31 of them: the last rows as the first."""
    from samnerf_amd import ops
    base = torch.randn((256, 65536), device="cuda", dtype=torch.bfloat16)
    x = base.repeat(150, 1)
    assert x.numel() > 1 << 31
    t, want = ops.top_logits(x, 16), ops.top_logits(base, 16)
    for a, b in zip(t, want):
        assert torch.equal(a[:256], b) and torch.equal(a[-256:], b)


# ---- loss ---------------------------------------------------------------------------------------------------------------------------
def loss64(z, ids, top, rest, T, keep=None):
    """(rows, counted) in float64 by autograd-able torch on the CPU."""
    R, V = z.shape
    u = z / T
    logq = torch.log_softmax(u, dim=1)
    rows, counted = [], []
    for r in range(R):
        on = ids[r] >= 0
        i, a = ids[r][on].long(), top[r][on] / T
        mass = torch.cat([a, rest[r:r + 1]]) if rest is not None else a
        if i.numel() == 0 or not bool((mass != -math.inf).any()):
            rows.append(z.new_zeros(()))
            counted.append(False)
            continue
        lp = torch.log_softmax(mass, dim=0)
        p = lp.exp()
        live = p[:i.numel()] > 0
        row = (p[:i.numel()][live] * (lp[:i.numel()][live] - logq[r][i[live]])).sum()
        if rest is not None and p[-1] > 0:
            other = torch.ones(V, dtype=torch.bool)
            other[i] = False
            row = row + p[-1] * (lp[-1] - torch.logsumexp(logq[r][other], dim=0))
        rows.append(row * T * T)
        counted.append(True)
    return torch.stack(rows), torch.tensor(counted)


def make(R, V, K, dtype, seed, empty=0.2, with_rest=True, T=1.0):
    g = torch.Generator().manual_seed(seed)
    teacher = 3 * torch.randn((R, V), generator=g)
    z = (0.6 * teacher + 1.5 * torch.randn((R, V), generator=g)).to(dtype)
    top, ids = torch.topk(teacher, K, dim=1)
    rest = torch.logsumexp(teacher.scatter(1, ids, -math.inf) / T, dim=1) if with_rest else None
    ids = ids.to(torch.int32)
    if empty:
        ids[torch.rand((R, K), generator=g) < 0.1] = -1
        ids[torch.rand((R,), generator=g) < empty] = -1
    return z, ids, top.to(dtype), rest


def check_loss(z, ids, top, rest, T, weight=1.0, gscale=1.0):
    """Loss per row and its gradient, for reductions none, mean and sum."""
    from samnerf_amd import ops
    R, V = z.shape
    zd = z.double().requires_grad_(True)
    rows, counted = loss64(zd, ids, top.double(), rest.double() if rest is not None else None, T)
    gr = torch.linspace(0.5, 1.5, R, dtype=torch.float64)
    (want,) = torch.autograd.grad((rows * gr).sum(), zd, allow_unused=True) if bool(counted.any()) else (None,)
    want = (want if want is not None else torch.zeros_like(zd)).detach() * weight
    rows = rows.detach() * weight
    dev = lambda t: t.cuda() if t is not None else None  # noqa: E731
    x = z.cuda().requires_grad_(True)
    got = ops.top_logits_distill_loss(x, dev(ids), dev(top), rest=dev(rest), temperature=T, weight=weight, reduction="none")
    (dx,) = torch.autograd.grad(got, x, gr.float().cuda())
    # A row's loss is a sum of p (log p - log q) with sum p = 1: each logarithm is off by at most 2^-24 times the size of its terms (logits
    # over T, their maxima, log-sums), the sums by 2^-24 a level (tree and at most 128 terms a thread).
    fin = lambda t: torch.nan_to_num(t.double().abs(), nan=0.0, posinf=0.0, neginf=0.0)  # noqa: E731
    size = (fin(z).max(1).values + fin(top).max(1).values) / T + math.log(V + 1.0) + 1.0
    tol = weight * T * T * U * 160 * size
    g64 = got.detach().cpu().double()
    ok = (g64 == rows) | ((g64 - rows).abs() <= tol)
    assert bool(ok.all()), (g64[~ok], rows[~ok])
    # dz = gs (q - p - p_rest q / q_rest): q, p and q / q_rest are exponentials of differences whose error is that of the logarithms above
    logq = torch.log_softmax(z.double() / T, dim=1)
    q = logq.exp()
    named = torch.zeros((R, V + 1), dtype=torch.bool).scatter_(1, torch.where(ids >= 0, ids.long(), V), True)[:, :V]
    mass = torch.where(named, torch.zeros_like(q), q)
    share = mass / mass.sum(1, keepdim=True).clamp_min(1e-300) if rest is not None else torch.zeros_like(q)
    part = weight * T * gr[:, None] * (q + share + named.double())
    fi = torch.finfo(z.dtype)
    gtol = part * U * 160 * size[:, None] + want.abs() * fi.eps / 2 * 1.01 + fi.smallest_normal * fi.eps
    d = dx.cpu().double()
    bad = (d - want).abs() > gtol
    assert not bool(bad.any()), ((d - want).abs()[bad].max(), gtol[bad].max(), int(bad.sum()))
    n = max(1, int(counted.sum()))
    for reduction, div in (("mean", n), ("sum", 1)):
        x = z.cuda().requires_grad_(True)
        loss = ops.top_logits_distill_loss(x, dev(ids), dev(top), rest=dev(rest), temperature=T, weight=weight, reduction=reduction)
        (dx2,) = torch.autograd.grad(loss, x, torch.tensor(gscale, device="cuda"))
        # (a sum over R rows: R / 1024 terms a thread and a tree)
        assert abs(float(loss) - float(rows.sum()) / div) <= float(tol.sum()) / div + U * (12 + R / 1024) * float(rows.abs().sum()) / div
        scaled = want / gr[:, None] * gscale / div
        t2 = gtol / gr[:, None] * gscale / div + scaled.abs() * 4 * U + fi.smallest_normal * fi.eps
        assert not bool(((dx2.cpu().double() - scaled).abs() > t2).any())
    return got, dx


LOSS_SIZES = [(1, 1, 1), (3, 2, 1), (4, 5, 5), (9, 64, 3), (33, 192, 8), (6, 257, 200), (5, 1003, 16), (2, 2048, 64), (7, 4100, 33),
              (1, 32000, 8), (3, 70000, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("R,V,K", LOSS_SIZES)
def test_distill_vs_reference(R, V, K, with_rest, dtype):
    for T, weight in ((1.0, 1.0), (2.5, 0.3)):
        check_loss(*make(R, V, K, dtype, R + V + K, with_rest=with_rest, T=T), T, weight, gscale=0.7)


@pytest.mark.parametrize("with_rest", [False, True])
def test_distill_gradient_vs_differences(with_rest):
    """Central differences of the kernel's own loss along random directions: step h, third-order term h^2 / 6 |d^3|, rounding U |loss| / h."""
    from samnerf_amd import ops
    z, ids, top, rest = make(6, 80, 7, torch.float32, 3, with_rest=with_rest, T=1.5)
    a = [t.cuda() if t is not None else None for t in (ids, top, rest)]
    f = lambda x: ops.top_logits_distill_loss(x, a[0], a[1], rest=a[2], temperature=1.5, reduction="sum")  # noqa: E731
    x = z.cuda().requires_grad_(True)
    (g,) = torch.autograd.grad(f(x), x)
    gen = torch.Generator().manual_seed(1)
    h = 2.0 ** -6
    for _ in range(5):
        d = torch.randn(z.shape, generator=gen).cuda()
        diff = float(f(z.cuda() + h * d).double() - f(z.cuda() - h * d).double()) / (2 * h)
        # the third derivative of log-sum-exp along d is at most (max d - min d)^3 / T^3 per row and term (two terms with rest)
        third = float(((d.max(1).values - d.min(1).values) ** 3).sum()) / 1.5 * 2
        assert abs(diff - float((g * d).sum())) <= h * h / 6 * third + 160 * U * 20 * 6 * 2.25 / h


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_rest", [False, True])
def test_distill_masks_and_extremes(with_rest, dtype):
    z, ids, top, rest = make(10, 300, 6, dtype, 11, empty=0, with_rest=with_rest)
    low = torch.finfo(dtype).min
    ids[0] = -1                                     # no entry
    top[1] = -math.inf                              # a teacher without mass (with rest: all of it there)
    z[2, 100:] = -math.inf                          # masked student places, named ones among the others
    ids[2] = torch.arange(6, dtype=torch.int32)
    z[3, 50:60] = low
    top[4, 3:] = -math.inf                          # entries without mass
    top[5, 2:] = low
    ids[6] = ids[6, 0].clone()                      # one place named six times
    ids[7, 1] = ids[7, 0]
    z[8] = 0.0
    z[9, 7:] = -200.0                               # all of the student's mass on few places, all of them named
    ids[9] = torch.arange(6, dtype=torch.int32)
    for T in (1.0, 3.0):
        check_loss(z, ids, top, rest, T)


@pytest.mark.parametrize("with_rest", [False, True])
def test_distill_infinite_and_bad_rows(with_rest):
    """Zero probability where the teacher has mass: an infinite loss, finite gradient; NaN logits and ids past the end: NaN; the rows beside
    them are as ever, and a row without a target is 0 whatever its logits are."""
    from samnerf_amd import ops
    z, ids, top, rest = make(6, 90, 5, torch.float32, 5, empty=0, with_rest=with_rest)
    good = check_loss(z, ids, top, rest, 1.0)
    z[0, ids[0, 0].long()] = -math.inf
    z[1, 3] = math.nan
    ids[2, 1] = 90
    ids[3] = -7
    z[3] = math.nan
    ids[4, 2] = 2 ** 31 - 1
    x = z.cuda().requires_grad_(True)
    r = ops.top_logits_distill_loss(x, ids.cuda(), top.cuda(), rest=rest.cuda() if with_rest else None, reduction="none")
    (g,) = torch.autograd.grad(r, x, torch.ones_like(r))
    assert float(r[0]) == math.inf and bool(torch.isfinite(g[0]).all())
    assert abs(float(g[0].double().sum())) <= 300 * U  # q and p both sum to 1
    for i in (1, 2, 4):
        assert math.isnan(float(r[i])) and bool(torch.isnan(g[i]).any())
    assert float(r[3]) == 0.0 and bool((g[3] == 0).all())
    assert torch.equal(r[5], good[0][5]) and bool(torch.isfinite(g[5]).all())
    assert bool(torch.isnan(g[2]).all()) and bool(torch.isnan(g[4]).all())


def test_distill_without_any_target():
    from samnerf_amd import losses, ops
    x = torch.randn((5, 40), device="cuda", requires_grad=True)
    ids, top = torch.full((5, 3), -1, dtype=torch.int64, device="cuda"), torch.randn((5, 3), device="cuda")
    loss = ops.top_logits_distill_loss(x, ids, top)
    (g,) = torch.autograd.grad(loss, x)
    assert float(loss) == 0.0 and bool((g == 0).all())
    e = torch.zeros((0, 40), device="cuda", requires_grad=True)
    loss = losses.TopLogitsDistillLoss()(e, ops.top_logits(e, 3))
    (g,) = torch.autograd.grad(loss, e)
    assert float(loss) == 0.0 and g.shape == (0, 40)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_layouts(dtype):
    """Leading dimensions, 64-bit ids, strided and misaligned rows, an expanded student, another float type for the teacher."""
    from samnerf_amd import ops
    z, ids, top, rest = (t.cuda() for t in make(12, 101, 5, dtype, 2, empty=0.2))

    def both(student, i=ids, t=top, r=rest):
        x = student.detach().requires_grad_(True)
        loss = ops.top_logits_distill_loss(x, i, t, rest=r, temperature=2.0)
        return loss.detach(), torch.autograd.grad(loss, x)[0]

    want, g = both(z)
    a, ga = both(z.view(3, 4, 101), ids.view(3, 4, 5).long(), top.view(3, 4, 5), rest.view(3, 4))
    assert torch.equal(a, want) and torch.equal(ga.view(12, 101), g)
    for off, extra in ((0, 3), (3, 8), (1, 27)):
        buf = torch.full((off + 12 * (101 + extra),), math.nan, dtype=dtype, device="cuda")
        s = torch.as_strided(buf, (12, 101), (101 + extra, 1), off)
        s.copy_(z)
        b, gb = both(s)
        # another alignment deals the row's places to other threads: sums in another order
        assert abs(float(b) - float(want)) <= 200 * U * abs(float(want)) + 200 * U
        assert float((gb.double() - g.double()).abs().max()) <= 4 * torch.finfo(dtype).eps * float(g.double().abs().max())
    c, gc = both(z, ids.t().contiguous().t(), top.t().contiguous().t())
    assert torch.equal(c, want) and torch.equal(gc, g)
    d, gd = both(z, ids, top.float())
    assert torch.equal(d, want) and torch.equal(gd, g)  # the same values in a wider type
    row = z[:1].clone().requires_grad_(True)
    loss = ops.top_logits_distill_loss(row.expand(12, 101), ids, top, rest=rest, temperature=2.0)
    (ge,) = torch.autograd.grad(loss, row)
    _, full = both(z[:1].expand(12, 101).contiguous())
    assert ge.shape == (1, 101) and torch.equal(ge, full.sum(0, keepdim=True, dtype=dtype))
    v = z[1].clone().requires_grad_(True)
    assert ops.top_logits_distill_loss(v, ids[1], top[1], rest=rest[1], reduction="none").shape == ()


def test_distill_leaves_teacher_and_neighbours_alone():
    """No gradient for the teacher, no double backward, nothing written behind the gradient's last row, inputs unchanged."""
    from samnerf_amd import _opcore as C
    from samnerf_amd import ops
    z, ids, top, rest = (t.cuda() for t in make(7, 131, 4, torch.bfloat16, 2))
    copies = [t.clone() for t in (z, ids, top, rest)]
    x, t = z.clone().requires_grad_(True), top.float().requires_grad_(True)
    loss = ops.top_logits_distill_loss(x, ids, t, rest=rest)
    (g,) = torch.autograd.grad(loss, x, create_graph=True)
    assert t.grad is None
    with pytest.raises(RuntimeError):
        g.sum().backward()
    for a, b in zip(copies, (z, ids, top, rest)):
        assert torch.equal(a, b)
    R, V, K = 7, 131, 4
    f32 = dict(device="cuda", dtype=torch.float32)
    rows, cnt, stats, p = torch.empty(R, **f32), torch.empty(R, **f32), torch.empty(4 * R, **f32), torch.empty(R * K, **f32)
    dz = torch.full((R * V + 64,), 7.0, device="cuda", dtype=torch.bfloat16)
    st = C._stream()
    C._launch("snf_top_distill_fwd", C._p(z), 1, R, V, V, C._p(ids), 0, C._p(top), 1, C._p(rest), K, 1.0, 1.0, C._p(rows), C._p(cnt),
              C._p(stats), C._p(p), 0, None, None, None, 0, st)
    one = torch.ones(1, **f32)
    for off in (0, 1):  # rows of the gradient at the student's offsets from 16 bytes, and at others
        dz.fill_(7.0)
        C._launch("snf_top_distill_bwd", C._p(z), 1, R, V, V, C._p(ids), 0, K, 1.0, 1.0, C._p(one), 0, None, C._p(cnt), C._p(stats), C._p(p),
                  C._p(dz) + 2 * off, st)
        assert bool((dz[R * V + off:] == 7.0).all()) and bool((dz[:off] == 7.0).all())
        d = dz[off:off + R * V].view(R, V)
        (want,) = torch.autograd.grad(ops.top_logits_distill_loss(x, ids, top, rest=rest, reduction="sum"), x)
        assert torch.equal(d, want)


@pytest.mark.parametrize("R,V", [(64, 501), (2, 40000)])
def test_distill_repeats_streams_and_graphs(R, V):
    """The same bits again, on another stream, and from a replayed graph (forward and backward) with new inputs."""
    from samnerf_amd import ops
    K = 6
    sets = [[t.cuda() for t in make(R, V, K, torch.float32, s)] for s in range(3)]

    def step(z, ids, top, rest):
        x = z.detach().requires_grad_(True)
        loss = ops.top_logits_distill_loss(x, ids, top, rest=rest, temperature=2.0)
        return loss.detach(), torch.autograd.grad(loss, x)[0]

    want = [step(*s) for s in sets]
    again = step(*sets[0])
    assert torch.equal(again[0], want[0][0]) and torch.equal(again[1], want[0][1])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        out = step(*sets[1])
        t2 = ops.top_logits(sets[1][0], K)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(out[0], want[1][0]) and torch.equal(out[1], want[1][1])
    tops = [ops.top_logits(s[0], K) for s in sets]
    assert all(torch.equal(a, b) for a, b in zip(t2, tops[1]))
    held = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
        t2 = ops.top_logits(held[0], K)
    for i in (1, 2, 0):
        for a, b in zip(held, sets[i]):
            a.copy_(b)
        graph.replay()
        eager = step(*sets[i])  # eager work in between
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1]) and torch.equal(eager[1], want[i][1])
        assert all(torch.equal(a, b) for a, b in zip(t2, tops[i]))


def classes80(z, ids, top, rest, T):
    """Of rows whose ids are all entries: the teacher's mass per place [R, V] and of the rest [R], q [R, V], which are named, the rows' loss
    and its gradient.  Computed in 80 bits: at 1e-11 of a probability close to 1, 64 have four digits."""
    f80 = lambda t: np.asarray(t.double().numpy(), dtype=np.longdouble)  # noqa: E731
    R, V = z.shape
    row, i = np.arange(R)[:, None], ids.long().numpy()
    a = f80(top) / np.longdouble(T)
    if rest is not None:
        a = np.concatenate([a, f80(rest)[:, None]], 1)
    am = a.max(1, keepdims=True)
    lp = a - am - np.log(np.exp(a - am).sum(1, keepdims=True))
    u = f80(z) / np.longdouble(T)
    um = u.max(1, keepdims=True)
    logq = u - um - np.log(np.exp(u - um).sum(1, keepdims=True))
    q = np.exp(logq)
    K = i.shape[1]
    p, named = np.zeros((R, V), np.longdouble), np.zeros((R, V), bool)
    np.add.at(p, (row, i), np.exp(lp[:, :K]))
    named[row, i] = True
    loss = (np.exp(lp[:, :K]) * (lp[:, :K] - logq[row, i])).sum(1)
    dz, pr = q - p, np.zeros(R, np.longdouble)
    if rest is not None:
        pr, other = np.exp(lp[:, -1]), (q * ~named).sum(1)
        loss += pr * (lp[:, -1] - np.log(other))
        dz -= np.where(named, 0, q) * (pr / other)[:, None]
    f64 = lambda a: torch.from_numpy(a.astype(np.float64))  # noqa: E731
    return f64(p), f64(pr), f64(q), torch.from_numpy(named), f64(loss * np.longdouble(T) ** 2), f64(dz * np.longdouble(T))


def check_digits(z, ids, top, rest, T):
    """Bounds that follow the result, also where a row's loss is small.  With d = log p - log q the loss is a sum of p d + q - p over the
    classes, and an error of d counts by p - q (where |d| > 1/2 by p or q, at most 2.6 |p - q|).  d is off by 8 steps of 2^-24 of the
    logits over T, and by what the sums are off: 64 places a lane in turn, a tree, some thousand parts joined by lanes, exponentials of
    exponents up to 30 (3 steps each): 160 + 90 steps.  Probabilities in p d + q - p: the same, at most 6 times the term."""
    from samnerf_amd import ops
    p, pr, q, named, rows, want = classes80(z, ids, top, rest, T)
    pn, qn = p.sum(1), (q * named).sum(1)
    qr = (q * ~named).sum(1)
    size = (z.double().abs().max(1).values + top.double().abs().max(1).values) / T + (rest.double().abs() if rest is not None else 0)
    steps = 250 + 8 * size
    apart = ((p - q) * named).abs().sum(1) + (pr - qr).abs()
    x = z.cuda().requires_grad_(True)
    got = ops.top_logits_distill_loss(x, ids.cuda(), top.cuda(), rest=rest.cuda() if rest is not None else None, temperature=T, reduction="none")
    (dx,) = torch.autograd.grad(got, x, torch.ones_like(got))
    off = (got.detach().cpu().double() - rows).abs()
    tol = T * T * U * steps * (2.6 * apart + 6 * rows / (T * T))
    assert bool((off <= tol).all()), (off / tol).max()
    # a place that is not named: (p_named - q_named) q / q_rest, the two sums off by `steps` of themselves, the exponential of (z - m) / T by
    # 3 steps of its exponent; then the result's own rounding
    fi = torch.finfo(z.dtype)
    share = q / qr.clamp_min(1e-300)[:, None]
    far = 3 * (z.double().max(1, keepdim=True).values - z.double()) / T + 8
    gtol = T * share * U * ((steps * (pn + qn))[:, None] if rest is not None else steps[:, None] * qr[:, None]) + want.abs() * (U * far + fi.eps / 2 * 1.01)
    bad = ((dx.cpu().double() - want).abs() > gtol + fi.smallest_normal * fi.eps) & ~named
    assert not bool(bad.any()), ((dx.cpu().double() - want).abs() / gtol)[bad].max()
    return dx.cpu().double(), want, p, pr, q, named, steps


def grad_of_sum(z, ids, top, rest, T=1.0):
    from samnerf_amd import ops
    x = z.cuda().requires_grad_(True)
    loss = ops.top_logits_distill_loss(x, ids.cuda(), top.cuda(), rest=rest.cuda() if rest is not None else None, temperature=T, reduction="sum")
    return torch.autograd.grad(loss, x)[0].cpu().double()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [700, 5003, 40000, 100000])
@pytest.mark.parametrize("k", [1, 2, 8])
def test_distill_short_list_of_a_long_row(k, V, dtype):
    """The list holds little of the mass on both sides: rest against rest is a quotient of two numbers close to 1."""
    for T in (2.0, 4.0):
        for R in (1, 24):
            check_digits(*make(R, V, k, dtype, V + k + R, empty=0, T=T), T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("V,k", [(2, 1), (2, 2), (40, 7), (1003, 16), (9000, 130), (70000, 64)])
def test_distill_one_place_holds_nearly_all(V, k, with_rest, dtype):
    """One named place with nearly all of both masses, the last entry of the list or the first: its q - p is the others' p less their q, and
    the loss is of their size."""
    for T, gap in ((1.0, 12.0), (0.5, 4.0), (3.0, 45.0)):
        z, ids, top, rest = make(6, V, k, torch.float32, V + k, empty=0, with_rest=with_rest, T=T)
        if rest is not None and k == V:
            continue  # (nothing is left for the rest)
        up = gap + 2 * T * math.log(V)
        j = torch.arange(6) % k
        row = torch.arange(6)
        top[row, j] += up
        z[row, ids[row, j].long()] += up
        z, top = z.to(dtype), top.to(dtype)
        d, want, p, pr, q, named, steps = check_digits(z, ids, top, rest, T)
        others = 1 - torch.nn.functional.one_hot(ids[row, j].long(), V)
        of_others = ((p + q) * others).sum(1) + pr
        apart = torch.where(others == 0, of_others[:, None].expand(6, V), p + q)
        fi = torch.finfo(dtype)
        tol = T * U * steps[:, None] * apart + want.abs() * fi.eps / 2 * 1.01 + fi.smallest_normal * fi.eps
        bad = ((d - want).abs() > tol) & named
        assert not bool(bad.any()), ((d - want).abs() / tol)[bad].max()


def test_distill_place_named_twice_holds_nearly_all():
    """Two entries for the heavy place, first and last of the list: their masses add up, the place counts once for the student."""
    for with_rest in (False, True):
        z, ids, top, rest = make(4, 300, 6, torch.float32, 9, empty=0, with_rest=with_rest)
        ids[:, 5] = ids[:, 0]
        top[:, 0] += 14.0
        top[:, 5] = top[:, 0] - 1.0
        z[torch.arange(4), ids[:, 0].long()] += 16.0
        check_loss(z, ids, top, rest, 1.0)
        p, pr, q, named, _, want = classes80(z, ids, top, rest, 1.0)
        d = grad_of_sum(z, ids, top, rest)
        heavy = torch.nn.functional.one_hot(ids[:, 0].long(), 300).bool()
        of_others = ((p + q) * ~heavy).sum(1) + pr
        steps = 250 + 8 * (z.double().abs().max(1).values + top.double().abs().max(1).values + (0 if rest is None else rest.double().abs()))
        assert bool(((d - want).abs()[heavy] <= U * steps * of_others).all())  # (as check_digits)


@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("V", [50, 1003, 40000])
def test_distill_gradient_entries_far_below_the_maximum(V, with_rest):
    """Two places that are not named have gradients in the ratio exp((z_v - z_w) / T): entries far below the largest keep their digits.  An
    entry is off by a step for the exponential's own rounding (1 ulp is 2 steps of 2^-24), one each for 1 + the rest of the exponent, its
    product, f and the product with it; two of them by 12, and the rest's own rounding is of second order.  (A temperature is a float32: 2.7
    as a double is 1.8e-8 beside it, 60 times that in the exponent is 18 steps.)"""
    for T in (0.5, 1.0, float(np.float32(2.7))):
        z, ids, top, rest = make(5, V, 4, torch.float32, V, empty=0, with_rest=with_rest, T=T)
        z = z + 7.3
        z[:, ::3] -= torch.rand((5, z[:, ::3].shape[1]), generator=torch.Generator().manual_seed(V)) * 60.0 * T
        d = grad_of_sum(z, ids, top, rest, T)
        masked = z.double().scatter(1, ids.long(), -math.inf)
        at = masked.argmax(1, keepdim=True)
        want = torch.exp((masked - masked.gather(1, at)) / T)
        seen = want > 1e-30  # (below: too near to the smallest normal number)
        off = (d / d.gather(1, at) - want).abs() / want
        assert bool((d.gather(1, at) != 0).all()) and float(off[seen].max()) <= 12 * U, float(off[seen].max()) / U


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_distill_second_derivative_is_refused(reduction):
    """With create_graph the gradient is what it is without, and part of the graph: a term of a loss that holds it cannot be dropped."""
    from samnerf_amd import ops
    z, ids, top, rest = (t.cuda() for t in make(6, 90, 5, torch.float32, 4, empty=0))
    views = (lambda x: x, lambda x: x.view(2, 3, 90), lambda x: x[:1].expand(6, 90), lambda x: x.t().contiguous().t())
    for view in views:
        x = z.clone().requires_grad_(True)
        s = view(x)
        lead = s.shape[:-1]

        def loss_of():
            return ops.top_logits_distill_loss(s, ids.view(*lead, 5), top.view(*lead, 5), rest=rest.view(lead), reduction=reduction).sum()

        (want,) = torch.autograd.grad(loss_of(), x)
        loss = loss_of()
        (g,) = torch.autograd.grad(loss, x, create_graph=True)
        assert torch.equal(g, want) and not want.requires_grad and g.requires_grad
        for what in (lambda: loss + g.pow(2).sum(), lambda: g.sum()):
            with pytest.raises(RuntimeError, match="no second derivative"):
                what().backward()
            loss = loss_of()
            (g,) = torch.autograd.grad(loss, x, create_graph=True)
    scale = torch.ones((), device="cuda", requires_grad=True)  # an incoming gradient that requires one
    x = z.clone().requires_grad_(True)
    loss = scale * ops.top_logits_distill_loss(x, ids, top, rest=rest)
    (g,) = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), scale)


def test_distill_student_written_after_the_call():
    """Where the call has copied the student (its rows are not contiguous), writing the original afterwards changes nothing; a student that
    is read in place again by the backward pass must not be written."""
    from samnerf_amd import ops
    z, ids, top, rest = (t.cuda() for t in make(6, 90, 5, torch.float32, 4, empty=0))
    for view in (lambda x: x.t().contiguous().t(), lambda x: x.view(2, 3, 90).permute(0, 2, 1).contiguous().permute(0, 2, 1)):
        x = z.clone().requires_grad_(True)
        s = view(x)
        lead = s.shape[:-1]
        args = (ids.view(*lead, 5), top.view(*lead, 5), rest.view(lead))
        (want,) = torch.autograd.grad(ops.top_logits_distill_loss(s, *args), x)
        s = view(x)
        loss = ops.top_logits_distill_loss(s, *args)
        with torch.no_grad():
            s.zero_()
        assert torch.equal(torch.autograd.grad(loss, x)[0], want)
    x = z.clone().requires_grad_(True)
    s = x * 1.0
    loss = ops.top_logits_distill_loss(s, ids, top, rest)
    with torch.no_grad():
        s.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("T,weight", [(1.7e19, 1.0), (2e-19, 1.0), (1e15, 1e-30), (1e-15, 1e30), (2.0, 0.0)])
def test_distill_at_the_ends_of_the_scale(T, weight, with_rest):
    """Temperatures and weights whose weight T^2 is just inside float32, logits of the temperature's size: the loss and the gradient of the
    same rows at T near 1, scaled."""
    z, ids, top, rest = make(5, 60, 4, torch.float32, 8, empty=0, with_rest=with_rest)
    # logits at the temperature's size; the rest has been divided by it
    k = 2.0 ** round(math.log2(T))
    Tk = T / k
    from samnerf_amd import ops
    x = (z * k).cuda().requires_grad_(True)
    a = dict(rest=rest.cuda() if with_rest else None, reduction="none")
    got = ops.top_logits_distill_loss(x, ids.cuda(), (top * k).cuda(), temperature=T, weight=weight, **a)
    (g,) = torch.autograd.grad(got, x, torch.ones_like(got))
    y = z.cuda().requires_grad_(True)
    want = ops.top_logits_distill_loss(y, ids.cuda(), top.cuda(), temperature=Tk, weight=1.0, **a)
    (h,) = torch.autograd.grad(want, y, torch.ones_like(want))
    # powers of two move nothing but the scale: T = k Tk to a rounding of T (exponents up to 20, as many steps), weight T^2 and weight T to one
    scale = weight * T * T / (Tk * Tk)
    over = want.double() * scale > torch.finfo(torch.float32).max  # a loss that no float32 holds: infinite
    assert bool(torch.isfinite(g).all()) and torch.equal(torch.isinf(got), over) and not bool(torch.isnan(got).any())
    got = torch.where(over, want.double() * scale, got.double())
    assert bool(((got - want.double() * scale).abs() <= 60 * U * abs(scale) * (want.double().abs() + Tk * Tk)).all())
    assert bool(((g.double() - h.double() * (weight * k)).abs() <= 60 * U * weight * k * Tk * 2).all())


def test_refusals_at_the_library():
    from samnerf_amd import _lib
    from samnerf_amd import _opcore as C
    x = torch.zeros((4, 64), device="cuda")
    i = torch.zeros((4, 64), device="cuda", dtype=torch.int32)
    ok = dict(x=C._p(x), dtype=0, R=4, V=64, ld=64, k=3, T=1.0)
    for bad in (dict(k=0), dict(k=65), dict(T=0.0), dict(T=float("nan")), dict(dtype=3), dict(ld=63), dict(R=-1), dict(V=0), dict(x=None),
                dict(R=1, V=1000001, ld=1000001)):
        a = {**ok, **bad}
        with pytest.raises(_lib.SnfError):
            C._launch("snf_top_logits", a["x"], a["dtype"], a["R"], a["V"], a["ld"], a["k"], a["T"], C._p(i), C._p(x), C._p(x), None, 0, C._stream())
    with pytest.raises(_lib.SnfError, match="workspace"):  # one long row is taken in parts
        C._launch("snf_top_logits", C._p(x), 0, 1, 200000, 200000, 3, 1.0, C._p(i), C._p(x), C._p(x), None, 0, C._stream())
    with pytest.raises(_lib.SnfError, match="workspace"):
        C._launch("snf_top_distill_fwd", C._p(x), 0, 1, 200000, 200000, C._p(i), 0, C._p(x), 0, None, 3, 1.0, 1.0, C._p(x), C._p(x), C._p(x),
                  C._p(x), 0, None, None, None, 0, C._stream())
    with pytest.raises(_lib.SnfError):
        C._launch("snf_top_distill_fwd", C._p(x), 0, 4, 64, 64, C._p(i), 0, C._p(x), 0, None, 257, 1.0, 1.0, C._p(x), C._p(x), C._p(x), C._p(x),
                  0, None, None, None, 0, C._stream())
    with pytest.raises(_lib.SnfError):
        C._launch("snf_top_distill_bwd", C._p(x), 0, 4, 64, 64, C._p(i), 0, 3, 1.0, 1.0, None, 0, None, C._p(x), C._p(x), C._p(x), C._p(x),
                  C._stream())
