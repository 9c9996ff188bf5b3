"""CPU tests of the top-logits operators: what they refuse before any launch."""
import pytest
import torch


def _args(lead=(4,), V=20, K=3):
    return torch.zeros(lead + (V,)), torch.zeros(lead + (K,), dtype=torch.int32), torch.zeros(lead + (K,)), torch.zeros(lead)


def test_top_logits_refusals():
    from samnerf_amd import ops
    x = torch.zeros((4, 20))
    for bad in (dict(k=0), dict(k=21), dict(k=3, temperature=0.0), dict(k=3, temperature=float("nan")), dict(k=3, temperature=float("inf")),
                dict(k=3, temperature=-1.0)):
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
