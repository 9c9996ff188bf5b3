"""A teacher's top logits and the distillation loss that reads them (csrc/distill.hip); `samnerf_amd.ops` re-exports everything here."""
from __future__ import annotations

from ctypes import c_float
from typing import NamedTuple, Optional

import torch

from ._opcore import DTYPE_CODE, _dev, _L, _launch, _p, _rows, _stream_on

__all__ = ["TopLogits", "top_logits", "top_logits_distill_loss", "TOP_LOGITS_MAX_K", "TOP_LOGITS_MAX_V"]

TOP_LOGITS_MAX_K = 256
TOP_LOGITS_MAX_V = 1000000  # SNF_TOP_MAX_V

_REDUCTIONS = ("mean", "sum", "none")


class TopLogits(NamedTuple):
    """What a teacher's answer is stored as: ids [..., k] int32 and logits [..., k], largest first, and rest [...] float32, the log-sum-exp
    of logit / temperature over all the other places (-inf where there are none)."""
    ids: torch.Tensor
    logits: torch.Tensor
    rest: torch.Tensor


def _temperature(t) -> float:
    t = float(t)
    if not 2.0 ** -126 <= t <= 3.4028234663852886e38:
        raise ValueError(f"temperature: a positive normal float32 expected, got {t}")
    return c_float(t).value


def _weight(w, t: float) -> float:
    # the loss is a row's divergence times weight T^2: 0, or within float32's normal numbers
    w = float(w)
    scale = abs(c_float(w).value) * t * t
    if w != 0.0 and not (2.0 ** -126 <= abs(w) < 2.0 ** 128 and 2.0 ** -126 <= scale < 2.0 ** 128):
        raise ValueError(f"weight, temperature: weight and weight T^2 have to be 0 or normal float32 numbers, got {w} and {scale}")
    return w


def _logits(t, name: str) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype not in DTYPE_CODE:
        raise TypeError(f"{name}: float32, bfloat16 or float16 expected, got {getattr(t, 'dtype', type(t))}")
    if t.dim() < 1 or not 1 <= t.shape[-1] <= TOP_LOGITS_MAX_V:
        raise ValueError(f"{name}: rows of 1 to {TOP_LOGITS_MAX_V} logits expected, got {tuple(t.shape)}")
    if t.numel() // t.shape[-1] >= 1 << 31:  # (the library counts rows in 32 bits)
        raise ValueError(f"{name}: fewer than 2^31 rows expected, got {tuple(t.shape)}")


def _rows_in_place(t: torch.Tensor) -> bool:
    """Whether `_rows(t)` is a view."""
    if t.is_contiguous():
        return True
    try:
        m = t.detach().view(-1, t.shape[-1]) if t.dim() != 2 else t
    except RuntimeError:
        return False
    return not (m.shape[1] > 1 and m.stride(1) != 1 or m.shape[0] > 1 and m.stride(0) < m.shape[1])


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty((nbytes // 8,), device=device, dtype=torch.int64) if nbytes else None


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The k largest of logits [..., V] with their places and the log-sum-exp of logits / temperature over all other places.  Equal logits
    come in the order of their places; a NaN counts as larger than everything.  k <= min(V, 256)."""
    _logits(logits, "logits")
    V, k = int(logits.shape[-1]), int(k)
    if not 1 <= k <= min(V, TOP_LOGITS_MAX_K):
        raise ValueError(f"top_logits: k={k} is not in 1 .. {min(V, TOP_LOGITS_MAX_K)}")
    t = _temperature(temperature)
    di, dev = _dev(logits, "logits"), logits.device
    lead = logits.shape[:-1]
    ids = torch.empty(lead + (k,), device=dev, dtype=torch.int32)
    vals = torch.empty(lead + (k,), device=dev, dtype=logits.dtype)
    rest = torch.empty(lead, device=dev, dtype=torch.float32)
    R = rest.numel()
    if R:
        x, ld = _rows(logits.detach() if logits.requires_grad else logits)
        code = DTYPE_CODE[x.dtype]
        nbytes = int(_L().snf_top_logits_workspace_bytes(R, V, k, code))
        ws = _workspace(nbytes, dev)
        _launch("snf_top_logits", _p(x), code, R, V, ld, k, t, _p(ids), _p(vals), _p(rest), _p(ws), nbytes, _stream_on(di),
                units=float(R * V * x.element_size()))
    return TopLogits(ids, vals, rest)


class _OnceDifferentiable(torch.autograd.Function):
    # the gradient as a function of what it depends on, for create_graph: asking for its derivative is refused, not answered with nothing
    @staticmethod
    def forward(ctx, student, g, first):
        return _TopDistill._gradient(first, g)

    @staticmethod
    def backward(ctx, g):
        raise RuntimeError("top_logits_distill_loss has no second derivative (its gradient was differentiated)")


class _TopDistill(torch.autograd.Function):
    # one buffer of floats: stats [R, 2], diff [R, K], counted [R], the divisor, rows [R] (unless they are the result)
    @staticmethod
    def forward(ctx, student, ids, logits, rest, temperature: float, weight: float, reduction: str):
        dev = student.device
        V, K = int(student.shape[-1]), int(ids.shape[-1])
        z, ld = _rows(student)
        ids, logits = ids.contiguous(), logits.contiguous()
        rest = rest.contiguous() if rest is not None else None
        R = z.shape[0]
        code = DTYPE_CODE[z.dtype]
        per_row = reduction == "none"
        saved = torch.empty((R * (4 + K) + 1,), device=dev, dtype=torch.float32)
        at = saved.data_ptr()
        counted, divisor, rows = at + 4 * R * (2 + K), at + 4 * R * (3 + K), at + 4 * R * (3 + K) + 4
        loss = torch.empty(student.shape[:-1] if per_row else (), device=dev, dtype=torch.float32)
        if R or not per_row:
            nbytes = int(_L().snf_top_distill_workspace_bytes(R, V, code))
            ws = _workspace(nbytes, dev)
            _launch("snf_top_distill_fwd", _p(z), code, R, V, ld, _p(ids), int(ids.dtype == torch.int64), _p(logits),
                    DTYPE_CODE[logits.dtype], _p(rest), K, temperature, weight, _p(loss) if per_row else rows, counted, at, at + 8 * R,
                    int(reduction == "mean"), None if per_row else _p(loss), divisor, _p(ws), nbytes, _stream_on(student.get_device()),
                    units=float(R * V * z.element_size()))
        ctx.args = (student.shape, R, V, ld, K, temperature, weight, per_row)
        ctx.save_for_backward(z, ids, saved, student)
        return loss

    @staticmethod
    def backward(ctx, g):
        dz = None
        if ctx.needs_input_grad[0]:
            dz = _OnceDifferentiable.apply(ctx.saved_tensors[3], g, ctx) if torch.is_grad_enabled() else _TopDistill._gradient(ctx, g)
        return dz, None, None, None, None, None, None

    @staticmethod
    def _gradient(ctx, g):
        z, ids, saved, _ = ctx.saved_tensors
        shape, R, V, ld, K, temperature, weight, per_row = ctx.args
        dz = torch.empty(shape, device=z.device, dtype=z.dtype)
        if R:
            if g.dtype != torch.float32 or not g.is_contiguous():
                g = g.to(torch.float32).contiguous()
            at = saved.data_ptr()
            counted, divisor = at + 4 * R * (2 + K), at + 4 * R * (3 + K)
            _launch("snf_top_distill_bwd", _p(z), DTYPE_CODE[z.dtype], R, V, ld, _p(ids), int(ids.dtype == torch.int64), K, temperature,
                    weight, _p(g), int(per_row), None if per_row else divisor, counted, at, at + 8 * R, _p(dz), _stream_on(z.get_device()),
                    units=float(2 * R * V * z.element_size()))
        return dz


def top_logits_distill_loss(student: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor, rest: Optional[torch.Tensor] = None,
                            temperature: float = 1.0, weight: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """weight * T^2 KL(teacher || student) from a teacher's top logits, with the student's gradient.

    student [..., V] logits; ids [..., K] (int32 / int64; a negative id is no entry) and logits [..., K] as `top_logits` returns them (any
    float type).  With rest [...] (float32, `top_logits` at the same temperature) the mass that the list leaves out is one class of its own,
    against the student's mass on all places that the ids do not name; without it the teacher's probabilities sum to 1 over the list.
    reduction "mean": over the rows with a target (a row without entries, or whose teacher has no mass, has none; no such row: 0); "sum";
    "none": [...] float32.  An id named twice counts twice for the teacher; an id >= V makes its row NaN.  The teacher's tensors get no
    gradient, and the gradient has no derivative of its own (a RuntimeError).  K <= 256.  (To capture the backward pass into a graph, let no eager graph of the same leaves live: autograd would
    accumulate on that graph's stream.)  weight and weight T^2 are 0 or normal float32 numbers."""
    _logits(student, "student")
    _logits(logits, "logits")
    t = _temperature(temperature)
    w = _weight(weight, t)
    lead = student.shape[:-1]
    if not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids: int32 or int64 expected, got {getattr(ids, 'dtype', type(ids))}")
    shape = ids.shape
    if len(shape) != student.dim() or shape[:-1] != lead or not 1 <= shape[-1] <= TOP_LOGITS_MAX_K:
        raise ValueError(f"ids: {tuple(lead)} rows of 1 to {TOP_LOGITS_MAX_K} expected, got {tuple(shape)}")
    if logits.shape != shape:
        raise ValueError(f"logits: {tuple(shape)} expected, got {tuple(logits.shape)}")
    if rest is not None:
        if not isinstance(rest, torch.Tensor) or rest.dtype != torch.float32:
            raise TypeError(f"rest: float32 expected, got {getattr(rest, 'dtype', type(rest))}")
        if rest.shape != lead:
            raise ValueError(f"rest: {tuple(lead)} expected, got {tuple(rest.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction: one of {_REDUCTIONS} expected, got {reduction!r}")
    di = _dev(student, "student")
    _dev(ids, "ids", di)
    _dev(logits, "logits", di)
    if logits.requires_grad:
        logits = logits.detach()
    if rest is not None:
        _dev(rest, "rest", di)
        if rest.requires_grad:
            rest = rest.detach()
    if not _rows_in_place(student):  # (copied here, not within: what is kept for the backward pass is then the copy alone)
        student = student.contiguous()
    return _TopDistill.apply(student, ids, logits, rest, t, w, reduction)
