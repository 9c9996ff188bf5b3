"""CPU tests of the top-logits operators: what they refuse before any launch."""
import pytest
import torch


def _args(lead=(4,), V=20, K=3):
    return torch.zeros(lead + (V,)), torch.zeros(lead + (K,), dtype=torch.int32), torch.zeros(lead + (K,)), torch.zeros(lead)


def test_top_logits_refusals():
    from samnerf_amd import ops
    x = torch.zeros((4, 20))
    for bad in (dict(k=0), dict(k=21), dict(k=3, temperature=0.0), dict(k=3, temperature=float("nan")), dict(k=3, temperature=float("inf")),
                dict(k=3, temperature=-1.0), dict(k=3, temperature=1e-39), dict(k=3, temperature=1e39)):
        with pytest.raises(ValueError):
            ops.top_logits(x, **bad)
    with pytest.raises(ValueError):
        ops.top_logits(torch.zeros((4, 300)), 257)
    with pytest.raises(ValueError):
        ops.top_logits(torch.zeros((4, 0)), 1)
    with pytest.raises(ValueError):
        ops.top_logits(torch.zeros((1, ops.TOP_LOGITS_MAX_V + 1)), 1)
    with pytest.raises(TypeError):
        ops.top_logits(x.double(), 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.top_logits(x, 2)


def test_distill_loss_refusals():
    from samnerf_amd import losses, ops
    z, ids, top, rest = _args()
    f = ops.top_logits_distill_loss
    with pytest.raises(TypeError):
        f(z.double(), ids, top)
    with pytest.raises(TypeError):
        f(z, ids.float(), top)
    with pytest.raises(TypeError):
        f(z, ids, top.double())
    with pytest.raises(TypeError):
        f(z, ids, top, rest=rest.double())
    for bad in ((z, ids[:3], top), (z, ids, top[:, :2]), (z[0], ids, top), (z, ids[:, :0], top[:, :0])):
        with pytest.raises(ValueError):
            f(*bad)
    wide = _args(K=257, V=300)
    with pytest.raises(ValueError):
        f(*wide[:3])
    for kw in (dict(rest=rest[:3]), dict(temperature=0), dict(reduction="batchmean")):
        with pytest.raises(ValueError):
            f(z, ids, top, **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        f(z, ids, top, rest=rest)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        losses.TopLogitsDistillLoss()(z, ops.TopLogits(ids, top, rest))


def test_the_library_refuses_before_any_launch():
    """Argument checks of the C entry points: host code, no device touched."""
    from samnerf_amd import _lib
    lib = _lib.load()
    p = 4096  # an aligned address that is never followed

    def refused(rc, word):
        assert rc == -1 and word in lib.snf_last_error(), (rc, lib.snf_last_error())

    ok = dict(x=p, dtype=0, R=4, V=64, ld=64, k=3, T=1.0, ids=p, logits=p, rest=p, ws=None, nbytes=0)

    def top(**kw):
        a = {**ok, **kw}
        return lib.snf_top_logits(a["x"], a["dtype"], a["R"], a["V"], a["ld"], a["k"], a["T"], a["ids"], a["logits"], a["rest"], a["ws"],
                                  a["nbytes"], None)

    for kw, word in ((dict(k=0), b"k=0"), (dict(k=65), b"k=65"), (dict(V=400, ld=400, k=257), b"k=257"), (dict(T=0.0), b"temperature"), (dict(T=1e-39), b"temperature"),
                     (dict(T=float("nan")), b"temperature"), (dict(dtype=3), b"dtype"), (dict(ld=63), b"overlap"), (dict(R=-1), b"sizes"),
                     (dict(V=1000001, ld=1000001), b"sizes"), (dict(x=None), b"null"), (dict(rest=None), b"null"),
                     (dict(V=200000, ld=200000), b"workspace"), (dict(R=2 ** 31 - 1, V=2, ld=2, k=1), b"too many")):
        refused(top(**kw), word)
    assert top(R=0, x=None) == 0
    n = lib.snf_top_logits_workspace_bytes(4, 200000, 3, 0)
    assert n == 4 * 8 * (-(-(200000 + 3) // 32)) and lib.snf_top_logits_workspace_bytes(4, 64, 3, 0) == 0

    def fwd(**kw):
        a = {**dict(z=p, dtype=0, R=4, V=64, ld=64, ids=p, top_dtype=0, K=3, T=1.0, stats=p, loss=None, divisor=None, nbytes=0), **kw}
        return lib.snf_top_distill_fwd(a["z"], a["dtype"], a["R"], a["V"], a["ld"], a["ids"], 0, p, a["top_dtype"], None, a["K"], a["T"], 1.0, p,
                                       p, a["stats"], p, 0, a["loss"], a["divisor"], None, a["nbytes"], None)

    for kw, word in ((dict(K=0), b"K=0"), (dict(K=257), b"K=257"), (dict(T=-1.0), b"temperature"), (dict(top_dtype=4), b"dtype"),
                     (dict(ld=8), b"overlap"), (dict(z=None), b"null"), (dict(stats=p + 4), b"aligned"), (dict(V=200000, ld=200000), b"workspace"),
                     (dict(loss=p), b"null")):
        refused(fwd(**kw), word)
    refused(lib.snf_top_distill_bwd(p, 0, 4, 64, 64, p, 0, 3, 1.0, 1.0, None, 0, None, p, p, p, p, None), b"null")
    refused(lib.snf_top_distill_bwd(p, 9, 4, 64, 64, p, 0, 3, 1.0, 1.0, p, 0, None, p, p, p, p, None), b"dtype")


def test_distill_loss_refuses_scales_outside_float32():
    """weight T^2 multiplies every row: where it is no normal float32 (and not 0) the loss would be infinite, NaN or 0 beside a finite
    gradient."""
    from samnerf_amd import _lib, ops
    z, ids, top, rest = _args()
    f = ops.top_logits_distill_loss
    lib = _lib.load()
    p = 4096  # an aligned address that is never followed

    def library(w, T):
        a = lib.snf_top_distill_fwd(None, 0, 4, 64, 64, None, 0, None, 0, None, 3, T, w, p, p, p, p, 0, None, None, None, 0, None)
        first = lib.snf_last_error()
        b = lib.snf_top_distill_bwd(None, 0, 4, 64, 64, None, 0, 3, T, w, None, 0, None, p, p, p, p, None)
        assert a == b == -1 and (b"weight" in first) == (b"weight" in lib.snf_last_error())
        return b"weight" in first  # (else: a null pointer)

    inside = ((1.0, 1.8e19), (1.0, 1.1e-19), (1e30, 1e4), (-1e-30, 1.1e-4), (0.0, 3e38), (0.0, 2e-38), (-2.0, 1.0), (3.4e38, 1.0), (1.2e-38, 1.0))
    outside = ((1.0, 1.9e19), (1.0, 1e-19), (1e30, 2e4), (-1e-30, 1e-4), (1e-40, 1e10), (1.0, 3e38), (float("nan"), 1.0), (float("inf"), 1.0),
               (3.5e38, 1.0))
    for w, T in inside:
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f(z, ids, top, rest=rest, temperature=T, weight=w)
        assert not library(w, T)
    for w, T in outside:
        with pytest.raises(ValueError, match="weight"):
            f(z, ids, top, rest=rest, temperature=T, weight=w)
        assert library(w, T)


def test_row_counts_past_32_bits_are_refused():
    """2^32 + 3 rows are not 3."""
    from samnerf_amd import ops
    n = 2 ** 32 + 3
    x = torch.zeros((1, 1)).expand(n, 1)
    with pytest.raises(ValueError, match="rows"):
        ops.top_logits(x, 1)
    with pytest.raises(ValueError, match="rows"):
        ops.top_logits_distill_loss(x, torch.zeros((1, 1), dtype=torch.int32).expand(n, 1), x)
