"""The operators of a quantised teacher and of distillation from its top logits: cases, plain forms, 64-bit values.

Four operators, in the order in which a training run uses them:

  quantize  rows -> microscaled 4-bit floats (blocks of 32 along the row, one power-of-two scale each) and back to the values they hold
  linear    act(rows W^T + bias) with both operands in that format: the teacher's (image encoder's) dense layers
  top       the k largest logits of a row, their places and the log-sum-exp of all the others: what a teacher's answer is stored as
  distill   KL(teacher's top logits || student) over rows with the student's gradient

`run` with `own` set makes the calls of `samnerf_amd.ops`; otherwise it computes the same in elementary torch operations in 32 bits.
"""
import math

import torch

own = False

_T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ACTS = ("none", "relu", "sigmoid", "gelu")
BLOCK = 32


def _ops():
    import samnerf_amd  # noqa: F401
    from samnerf_amd import ops
    return ops


# ---------------------------------------------------------------------------------------------------------------- cases
def _quantize(name, m, k, dtype, pad=0):
    return {"name": name, "op": "quantize", "m": m, "k": k, "dtype": dtype, "pad": pad}


def _linear(name, m, k, n, dtype, act="none", bias=True):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias}


def _top(name, rows, v, k, dtype, temperature=1.0):
    return {"name": name, "op": "top", "rows": rows, "v": v, "k": k, "dtype": dtype, "temperature": temperature}


def _distill(name, rows, v, k, dtype, temperature, rest, empty):
    return {"name": name, "op": "distill", "rows": rows, "v": v, "k": k, "dtype": dtype, "temperature": temperature, "rest": rest, "empty": empty}


def listed():
    return [
        # one token's row of the encoder's width: what a call costs
        _quantize("quantize_one_row", 1, 1280, "f32"),
        # the hidden rows between an encoder block's two MLP layers, one 64 x 64 token image
        _quantize("quantize_hidden", 4096, 5120, "bf16"),
        # one token through the first MLP layer
        _linear("linear_one_row", 1, 1280, 5120, "f32", "gelu"),
        # the windowed blocks' qkv layer: 25 windows of 14 x 14 tokens
        _linear("linear_qkv_windows", 4900, 1280, 3840, "f32"),
        # odd sizes in every direction
        _linear("linear_ragged", 333, 1003, 777, "f16", "relu", False),
        # four images' hidden rows through a square layer: bound by the matrix cores
        _linear("linear_large", 16384, 5120, 5120, "bf16"),
        # one answer over a long list of classes
        _top("top_one_row", 1, 32000, 8, "f32"),
        # a train step's rays over an odd number of classes
        _top("top_rays", 4096, 1003, 16, "f32", 2.0),
        # a long list for every ray
        _top("top_long", 4096, 65536, 64, "bf16"),
        # a patch of rays over the width of a feature head
        _distill("distill_patch", 256, 192, 8, "f32", 2.0, True, 0.1),
        # a train step's rays, the teacher's mass renormalised on its top logits, many rays without a target
        _distill("distill_rays", 4096, 1003, 16, "f32", 1.0, False, 0.3),
        # a long list for every ray, the rest of the mass in one class of its own
        _distill("distill_long", 4096, 65536, 64, "bf16", 2.0, True, 0.02),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "top", "distill", "distill"])
    dtype = rng.choice(list(_T))
    if op == "quantize":
        return _quantize(None, _log(rng, 1, 8192), _log(rng, 1, 5120), dtype, rng.choice([0, 0, 8, 5]))
    if op == "linear":
        return _linear(None, _log(rng, 1, 16384), _log(rng, 16, 5120), _log(rng, 1, 5120), dtype, rng.choice(_ACTS), rng.random() < 0.7)
    rows, most = _log(rng, 1, 8192), 4096 * 65536
    v = _log(rng, 2, max(2, min(131072, most // rows)))
    k = min(v, _log(rng, 1, 64))
    t = round(rng.uniform(0.5, 4.0), 2)
    if op == "top":
        return _top(None, rows, v, k, dtype, t)
    return _distill(None, rows, v, k, dtype, t, rng.random() < 0.5, rng.choice([0.0, 0.1, 0.5]))


# --------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows(g, m, k, dtype, pad=0):
    """Activations as the encoder has them: normalised rows whose channels differ in size by up to some tens."""
    scale = torch.exp(torch.randn((k,), generator=g, device="cuda"))
    x = torch.randn((m, k), generator=g, device="cuda").mul_(scale).to(_T[dtype])
    if pad:  # rows of a wider matrix
        wide = torch.empty((m, k + pad), device="cuda", dtype=_T[dtype])
        wide[:, :k] = x
        wide[:, k:] = float("nan")
        x = wide[:, :k]
    return x


def _inputs(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "quantize":
        return {"x": _rows(g, case["m"], case["k"], case["dtype"], case["pad"])}
    if op == "linear":
        k, n = case["k"], case["n"]
        d = {"x": _rows(g, case["m"], k, case["dtype"]), "w": torch.randn((n, k), generator=g, device="cuda") / math.sqrt(3.0 * k)}
        d["bias"] = 0.1 * torch.randn((n,), generator=g, device="cuda") if case["bias"] else None
        return d
    rows, v, k = case["rows"], case["v"], case["k"]
    teacher = torch.randn((rows, v), generator=g, device="cuda").mul_(3.0)
    if op == "top":
        return {"logits": teacher.to(_T[case["dtype"]])}
    student = torch.randn((rows, v), generator=g, device="cuda").mul_(1.5).add_(teacher, alpha=0.6).to(_T[case["dtype"]])
    top, ids = torch.topk(teacher, k, dim=1)
    others = teacher.scatter_(1, ids, float("-inf"))
    rest = torch.logsumexp(others / case["temperature"], dim=1) if case["rest"] else None
    ids = ids.to(torch.int32)
    if case["empty"]:
        ids[torch.rand((rows,), generator=g, device="cuda") < case["empty"]] = -1  # rows without a target
        ids[torch.rand((rows, k), generator=g, device="cuda") < 0.05] = -1  # shorter lists
    return {"student": student, "ids": ids, "top": top.to(_T[case["dtype"]]), "rest": rest}


def prepare(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "linear":  # a layer's weights are quantised once
        w = d.pop("w")
        d["weight"] = _ops().quantize_mxfp4(w) if own else _plain_quantize(w)
    if case["op"] == "distill" and own:
        d["student"].requires_grad_(True)
    return {"case": case, **d}


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_quantize(x):
    """The values of x [m, k] in microscaled 4-bit floats, as float32."""
    m, k = x.shape
    x = x.float()
    if k % BLOCK:
        x = torch.cat([x, x.new_zeros((m, BLOCK - k % BLOCK))], dim=1)
    b = x.reshape(m, -1, BLOCK)
    largest = b.abs().amax(dim=2, keepdim=True)
    e = torch.clamp(torch.frexp(largest).exponent - 3, min=-127)  # floor(log2(largest)) - 2
    e = torch.where(largest > 0, e, torch.full_like(e, -127))
    half = torch.div(e, 2, rounding_mode="floor")  # in two factors: 2^127 and 2^-127 are within the range, their like are not
    a = torch.ldexp(torch.ldexp(b.abs(), -half), half - e)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.clamp(torch.round(a / step) * step, max=6.0)  # round halves to even
    q = torch.ldexp(torch.ldexp(q, e - half), half)
    return torch.where(b < 0, -q, q).reshape(m, -1)[:, :k]


def _plain_act(y, act):
    if act == "relu":
        return torch.clamp(y, min=0.0)
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return y


def _plain_linear(s):
    y = _plain_quantize(s["x"]) @ s["weight"].t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return _plain_act(y, s["case"]["act"]).to(s["x"].dtype)


def _plain_top(s):
    x, k, t = s["logits"], s["case"]["k"], s["case"]["temperature"]
    v, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: the lowest place first
    others = v[:, k:].float()
    if others.shape[1]:
        m = others.amax(dim=1, keepdim=True)
        rest = (m / t).squeeze(1) + torch.log(torch.exp((others - m) / t).sum(dim=1))
    else:
        rest = torch.full((x.shape[0],), float("-inf"), device=x.device)
    return order[:, :k].to(torch.int32), v[:, :k].contiguous(), rest


def _plain_distill(s):
    t = s["case"]["temperature"]
    z, ids, top = s["student"].detach().float(), s["ids"].long(), s["top"].float()
    there = ids >= 0
    counted = there.any(dim=1)
    place = torch.where(there, ids, torch.zeros_like(ids))
    a = torch.where(there, top / t, torch.full_like(top, float("-inf")))
    if s["rest"] is not None:
        a = torch.cat([a, torch.where(counted, s["rest"], torch.zeros_like(s["rest"]))[:, None]], dim=1)
    else:
        a = torch.where(counted[:, None], a, torch.zeros_like(a))
    am = a.amax(dim=1, keepdim=True)
    counted = counted & (am.squeeze(1) != float("-inf"))  # a teacher without any mass is no target either
    am = torch.where(counted[:, None], am, torch.zeros_like(am))
    pe = torch.exp(a - am)
    ps = pe.sum(dim=1, keepdim=True)
    p, logp = pe / ps, (a - am) - torch.log(ps)  # the teacher's probabilities (the last column: everything else)
    zm = z.amax(dim=1, keepdim=True)
    u = (z - zm) / t
    e = torch.exp(u)
    total = e.sum(dim=1, keepdim=True)
    logq = u.gather(1, place) - torch.log(total)
    pk, logpk = p[:, :ids.shape[1]], logp[:, :ids.shape[1]]
    loss = torch.where(there & (pk > 0), pk * (logpk - logq), torch.zeros_like(pk)).sum(dim=1)
    grad = e / total
    if s["rest"] is not None:
        named = torch.zeros(z.shape, dtype=torch.bool, device=z.device)
        row, col = torch.nonzero(there, as_tuple=True)
        named[row, ids[row, col]] = True
        other = torch.where(named, torch.zeros_like(e), e)
        mass = other.sum(dim=1, keepdim=True)
        pr = p[:, -1:]
        loss = loss + torch.where(pr > 0, pr * (logp[:, -1:] - (torch.log(mass) - torch.log(total))), torch.zeros_like(pr)).squeeze(1)
        grad = grad - torch.where((pr > 0) & (other > 0), pr * other / mass, torch.zeros_like(other))
    grad = grad.scatter_add(1, place, torch.where(there, -pk, torch.zeros_like(pk)))
    n = torch.clamp(counted.sum(), min=1).float()
    loss = torch.where(counted, loss, torch.zeros_like(loss)).sum() * (t * t) / n
    grad = torch.where(counted[:, None], grad * (t / n), torch.zeros_like(grad))
    return loss, grad.to(s["student"].dtype)


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        if op == "quantize":
            return _plain_quantize(state["x"])
        return {"linear": _plain_linear, "top": _plain_top, "distill": _plain_distill}[op](state)
    ops = _ops()
    if op == "quantize":
        return ops.dequantize_mxfp4(ops.quantize_mxfp4(state["x"]))
    if op == "linear":
        return ops.linear_mxfp4(state["x"], state["weight"], state["bias"], act=ops.ACT_BY_NAME[case["act"]] if case["act"] != "gelu" else ops.ACT_GELU)
    if op == "top":
        return tuple(ops.top_logits(state["logits"], case["k"], temperature=case["temperature"]))
    z = state["student"]
    loss = ops.top_logits_distill_loss(z, state["ids"], state["top"], rest=state["rest"], temperature=case["temperature"])
    return loss.detach(), torch.autograd.grad(loss, z)[0]


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    op = case["op"]
    if op == "quantize":
        mk = case["m"] * case["k"]
        return {"bytes": mk * (size + 4), "flops": 4 * mk}
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        w = n * -(-k // BLOCK) * (BLOCK // 2 + 1)
        return {"bytes": m * k * size + w + (4 * n if case["bias"] else 0) + m * n * size, "flops": 2 * m * n * k}
    rows, v, k = case["rows"], case["v"], case["k"]
    if op == "top":
        return {"bytes": rows * (v * size + k * (size + 4) + 4), "flops": 4 * rows * v}
    return {"bytes": rows * (2 * v * size + k * (size + 4) + (4 if case["rest"] else 0)) + 4, "flops": 10 * rows * v}


# ------------------------------------------------------------------------------------------------------- values in 64 bits
def _exact_quantize(x):
    """Nearest of the eight magnitudes by comparison with the midpoints (a midpoint goes to the neighbour with the even code)."""
    m, k = x.shape
    pad = (-k) % BLOCK
    x = torch.nn.functional.pad(x.double(), (0, pad))
    b = x.view(m, (k + pad) // BLOCK, BLOCK)
    largest = b.abs().max(dim=2, keepdim=True).values
    power = torch.floor(torch.log2(torch.where(largest > 0, largest, torch.ones_like(largest)))) - 2
    scale = torch.pow(2.0, torch.clamp(power, min=-127.0))
    a = b.abs() / scale
    code = torch.zeros_like(a, dtype=torch.long)
    for i, mid in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a >= mid) if i % 2 else (a > mid)
    values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    return (torch.sign(b) * values[code] * scale).view(m, k + pad)[:, :k]


def exact(case, seed):
    d = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_quantize(d["x"])
    if op == "linear":
        y = torch.mm(_exact_quantize(d["x"]), _exact_quantize(d["w"]).t().contiguous())
        if d["bias"] is not None:
            y += d["bias"].double()
        act = case["act"]
        if act == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        elif act == "sigmoid":
            y = torch.reciprocal(1 + torch.exp(-y))
        elif act == "gelu":
            y = y * 0.5 * torch.erfc(-y / math.sqrt(2.0))
        return y
    t = float(case["temperature"])
    if op == "top":
        ids, logits, rest = [], [], []
        for x in d["logits"].split(512):
            # one whole number per entry: the logit's rank among all values first, the place second
            bits = x.float().contiguous().view(torch.int32).long()
            bits = torch.where(x.float() == 0, torch.zeros_like(bits), bits)
            rank = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
            place = torch.arange(x.shape[1], device=x.device)
            keep = torch.topk(rank * (1 << 20) - place, case["k"], dim=1, sorted=True).indices
            ids.append(keep.to(torch.int32))
            logits.append(x.double().gather(1, keep))
            rest.append(torch.logsumexp(x.double().div(t).scatter(1, keep, float("-inf")), dim=1))
        return torch.cat(ids), torch.cat(logits), torch.cat(rest)
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    grads = []
    has = (d["ids"] >= 0).any(dim=1)
    mass = torch.cat([d["top"].double().masked_fill(d["ids"] < 0, float("-inf"))] + ([d["rest"].double()[:, None]] if d["rest"] is not None else []), dim=1)
    has &= (mass != float("-inf")).any(dim=1)
    n = max(1, int(has.sum()))
    for lo in range(0, case["rows"], 1024):
        z = d["student"][lo:lo + 1024].double() / t
        ids, top = d["ids"][lo:lo + 1024].long(), d["top"][lo:lo + 1024].double() / t
        alive = ids >= 0
        weight = torch.zeros((z.shape[0], z.shape[1] + 1), dtype=torch.float64, device=z.device)  # a last column for what is not there
        ids = torch.where(alive, ids, torch.full_like(ids, z.shape[1]))
        lse = torch.logsumexp(top.masked_fill(~alive, float("-inf")), dim=1, keepdim=True)
        if d["rest"] is not None:
            lse = torch.logaddexp(lse, d["rest"][lo:lo + 1024].double()[:, None])
        lp = (top - lse).masked_fill(~alive, float("-inf"))
        weight.scatter_add_(1, ids, torch.exp(lp).nan_to_num(0.0).masked_fill(~alive, 0.0))
        weight = weight[:, :-1]
        logq = torch.log_softmax(z, dim=1)
        logq1 = torch.cat([logq, torch.zeros_like(logq[:, :1])], dim=1)
        row = torch.where(alive & (lp > float("-inf")), torch.exp(lp) * (lp - logq1.gather(1, ids)), torch.zeros_like(lp)).sum(dim=1)
        grad = torch.exp(logq) - weight
        if d["rest"] is not None:
            listed_ = torch.zeros((z.shape[0], z.shape[1] + 1), dtype=torch.bool, device=z.device).scatter_(1, ids, True)[:, :-1]
            lr = d["rest"][lo:lo + 1024].double() - lse.squeeze(1)
            others = logq.masked_fill(listed_, float("-inf"))
            lo_mass = torch.logsumexp(others, dim=1)
            some = lr > float("-inf")
            row = row + torch.where(some, torch.exp(lr) * (lr - lo_mass), torch.zeros_like(lr))
            grad = grad - torch.where(some[:, None] & ~listed_, torch.exp(lr[:, None] + others - lo_mass[:, None]), torch.zeros_like(grad))
        use = has[lo:lo + 1024]
        total += torch.where(use, row, torch.zeros_like(row)).sum()
        grads.append(torch.where(use[:, None], grad * (t / n), torch.zeros_like(grad)))
    return total * t * t / n, torch.cat(grads)
