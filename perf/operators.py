"""The label operators as they are measured: the product in 8-bit floating point that forms a row of class logits from a
row of features, the distillation loss that those logits learn from, and the draw of a label from them.

`run` computes each in its plain form (elementary torch operations) where `own` is false and makes the framework's calls
where it is true.  `exact` is the definition in 64 bits.

Definitions
  product   y = X8 W8^T + b.  X8 is x rounded to e4m3 in blocks of 128 consecutive columns of a row, W8 the weight in
            blocks of 128 x 128; a block's scale is the smallest power of two s with max|block| / s <= 448, held as the
            byte 127 + log2 s (a block of zeros: 127).  The gradients are the same product: dX = dY8 W8, with dY in blocks
            of 128 columns of a row, and dW = (dY^T)8 (X^T)8, both in blocks of 128 rows of a column; db = column sums.
  distill   loss_n = sum_j p_j (log p_j - log q_{i_j}), p = softmax of the teacher's values over T (the slots with an index
            in [0, V) alone), q = softmax of the student's row over T; a row without such a slot has loss 0 and gradient 0.
  draw      weights exp((z - max z) / T) of the top_k largest (ties: lowest index first), of those the smallest set whose
            share reaches top_p, of those the ones with weight >= min_p; the label is the first whose running sum, in the same
            order of falling weight, is over u times the total.  -1 where a row has nothing to draw.
"""
import math

import torch

own = False

BLOCK = 128
DEVICE = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---- the cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a training batch of rays against the object table's 64 labels: a call of a few microseconds
        dict(name="distill_batch", op="distill", form="grad", n=2048, v=64, k=8, type="fp32", teacher="fp32", t=1.0, gaps=False),
        # the same batch against an open vocabulary, inside a torch training loop
        dict(name="distill_autograd", op="distill", form="autograd", n=2048, v=32768, k=64, type="bf16", teacher="bf16", t=2.0, gaps=False),
        # the loss of a whole 640 x 480 frame, for a validation image
        dict(name="distill_frame", op="distill", form="loss", n=307200, v=64, k=4, type="fp32", teacher="fp16", t=1.0, gaps=False),
        # a ragged vocabulary whose teacher leaves slots and whole rows empty
        dict(name="distill_ragged", op="distill", form="grad", n=1023, v=30011, k=20, type="fp16", teacher="fp32", t=0.5, gaps=True),
        # one row of a large vocabulary: latency
        dict(name="draw_one", op="draw", n=1, v=131072, type="bf16", t=0.8, top_k=0, top_p=0.9, min_p=0.0, rows=False, masked=False),
        # an instance label for every ray of a frame
        dict(name="draw_frame", op="draw", n=307200, v=64, type="fp32", t=0.7, top_k=8, top_p=1.0, min_p=0.0, rows=False, masked=False),
        # a batch against an open vocabulary with every filter on
        dict(name="draw_batch", op="draw", n=2048, v=32768, type="bf16", t=1.0, top_k=50, top_p=0.95, min_p=0.02, rows=False, masked=False),
        # every row with settings of its own, masked labels, rows with nothing left
        dict(name="draw_rows", op="draw", n=257, v=30011, type="fp16", t=1.0, top_k=0, top_p=0.9, min_p=0.01, rows=True, masked=True),
        # the labels of a few picked pixels: the weight is all there is to read
        dict(name="linear_few", op="linear", form="weight8", m=4, n=32768, k=256, type="bf16", out="fp32", bias=False),
        # a hidden layer's 256 features on every ray of a frame
        dict(name="linear_frame", op="linear", form="weight8", m=307200, n=256, k=256, type="bf16", out="bf16", bias=True),
        # a large square product, where the matrix cores count
        dict(name="linear_large", op="linear", form="weight8", m=8192, n=8192, k=4096, type="bf16", out="bf16", bias=False),
        # a training step of a ragged layer: the forward product and all three gradients
        dict(name="linear_train", op="linear", form="train", m=16383, n=2056, k=520, type="bf16", out="bf16", bias=True),
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over the logarithm, odd as often as even."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["distill", "draw", "linear"])
    kind = rng.choice(sorted(TYPES))
    if op == "distill":
        v = _log(rng, 16, 131072)
        return dict(op=op, form=rng.choice(["grad", "autograd", "loss"]), n=_log(rng, 1, max(1, min(307200, 2048 * 32768 // v))), v=v,
                    k=_log(rng, 1, min(v, 128)), type=kind, teacher=rng.choice(sorted(TYPES)), t=rng.choice([0.5, 1.0, 2.0]),
                    gaps=rng.random() < 0.5)
    if op == "draw":
        v = _log(rng, 2, 131072)
        return dict(op=op, n=_log(rng, 1, max(1, min(307200, 2048 * 32768 // v))), v=v, type=kind, t=rng.choice([0.5, 0.8, 1.0, 1.5]),
                    top_k=rng.choice([0, 1, _log(rng, 1, v)]), top_p=rng.choice([1.0, 0.95, 0.5]), min_p=rng.choice([0.0, 0.02]),
                    rows=rng.random() < 0.3, masked=rng.random() < 0.5)
    form = rng.choice(["weight8", "weight8", "train"])
    k = _log(rng, 16, 8192)
    n = _log(rng, 1, min(32768, (1 << 26) // k))
    most = min(307200, (1 << 26) // max(n, k), (8192 * 8192 * 4096 // (4 if form == "train" else 1)) // (n * k))
    return dict(op=op, form=form, m=_log(rng, 1, max(1, most)), n=n, k=k, type=kind, out=rng.choice([kind, "fp32"]) if form != "train" else kind,
                bias=rng.random() < 0.5)


# ---- what a program has in hand before the call --------------------------------------------------------------------------

def _logits(g, n, v, dtype):
    """Rows of class scores: a broad floor and, in each row, a few labels that stand out."""
    z = torch.randn(n, v, device=DEVICE, generator=g) * 1.5
    few = min(v, 8)
    at = torch.randint(0, v, (n, few), device=DEVICE, generator=g)
    z.scatter_add_(1, at, torch.rand(n, few, device=DEVICE, generator=g) * 9.0)
    return z.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "distill":
        n, v, k = case["n"], case["v"], case["k"]
        s["student"] = _logits(g, n, v, TYPES[case["type"]])
        # the teacher agrees with the student in part: its slots are distinct labels, in no order
        first = torch.randint(0, v, (n, 1), device=DEVICE, generator=g)
        step = 2 * torch.randint(0, max(1, v // (2 * k)), (n, 1), device=DEVICE, generator=g) + 1
        index = (first + torch.arange(k, device=DEVICE) * torch.minimum(step, torch.tensor(max(1, v // k), device=DEVICE))) % v
        near = torch.gather(s["student"].float(), 1, index)
        s["teacher"] = (0.5 * near + 2.0 * torch.randn(n, k, device=DEVICE, generator=g)).to(TYPES[case["teacher"]])
        if case["gaps"]:
            off = torch.rand(n, k, device=DEVICE, generator=g) < 0.3
            off |= torch.rand(n, 1, device=DEVICE, generator=g) < 0.05
            index = torch.where(off, torch.full_like(index, -1), index)
        s["index"] = index.to(torch.int32)
        # a mean over the batch; half precision trains under a loss scale
        s["upstream"] = torch.rand(n, device=DEVICE, generator=g) * (2.0 / n) * (4096.0 if case["type"] == "fp16" else 1.0)
    elif case["op"] == "draw":
        n, v = case["n"], case["v"]
        s["logits"] = _logits(g, n, v, TYPES[case["type"]])
        if case["masked"]:
            off = torch.rand(n, v, device=DEVICE, generator=g) < 0.4
            off |= torch.rand(n, 1, device=DEVICE, generator=g) < 0.05
            s["logits"].masked_fill_(off, float("-inf"))
        s["u"] = torch.rand(n, device=DEVICE, generator=g)
        if case["rows"]:
            spread = torch.rand(4, n, device=DEVICE, generator=g)
            s["t"] = case["t"] * (0.5 + spread[0])
            s["top_k"] = (case["top_k"] * spread[1] + torch.where(spread[1] < 0.5, 0, 40)).to(torch.int32)
            s["top_p"] = 1 - (1 - case["top_p"]) * 2 * spread[2]
            s["min_p"] = case["min_p"] * spread[3]
        else:
            s.update({q: case[q] for q in ("t", "top_k", "top_p", "min_p")})
    else:
        m, n, k = case["m"], case["n"], case["k"]
        dtype = TYPES[case["type"]]
        # features after an activation, a few channels of them much larger than the rest
        x = torch.randn(m, k, device=DEVICE, generator=g)
        x = torch.where(x > 0, x, 0.01 * x) * torch.exp(torch.randn(k, device=DEVICE, generator=g))
        w = torch.randn(n, k, device=DEVICE, generator=g) * k ** -0.5
        s["x"], s["weight"] = x.to(dtype), w.to(dtype)
        s["bias"] = torch.randn(n, device=DEVICE, generator=g) if case["bias"] else None
        if case["form"] == "train":
            dy = torch.randn(m, n, device=DEVICE, generator=g) * torch.exp(torch.randn(m, 1, device=DEVICE, generator=g))
            s["dy"] = (dy * m ** -0.5).to(dtype)
        else:       # an inference program lays its weights out once
            s["weight8"] = _quantized(s["weight"], BLOCK)
            del s["weight"]
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------------

def _tiles(x, rows):
    """x (R, C) as (row blocks, rows, column blocks, 128), filled up with zeros."""
    r, c = x.shape
    up = torch.nn.functional.pad(x, (0, -c % BLOCK, 0, -r % rows))
    return up.reshape(up.shape[0] // rows, rows, up.shape[1] // BLOCK, BLOCK)


def _power(byte):
    """2 ** (byte - 127) for bytes of [1, 254], from the bits of the number: no rounding."""
    return (byte.int() << 23).view(torch.float32)


def _quantized(x, rows):
    """(values (R, C') in e4m3, scale bytes (R, B')): blocks of `rows` x 128; C' is C filled up to whole blocks and B' their
    number filled up to a multiple of 4 with 127."""
    t = _tiles(x.float(), rows)
    largest = t.abs().amax(dim=(1, 3), keepdim=True)
    half, power = torch.frexp(largest)                              # largest = half * 2^power, half in [0.5, 1)
    byte = (power - 9 + (half > 0.875) + 127).clamp(min=1)          # 448 = 0.875 * 2^9
    byte = torch.where(largest > 0, byte, torch.full_like(byte, 127))
    q = (t * _power(254 - byte)).reshape(-1, t.shape[2] * BLOCK)[:x.shape[0]].to(torch.float8_e4m3fn)
    byte = byte.expand(-1, rows, -1, -1).reshape(-1, t.shape[2])[:x.shape[0]]
    return q, torch.nn.functional.pad(byte, (0, -byte.shape[1] % 4), value=127).to(torch.uint8)


def _values(q, byte):
    """What (values, scale bytes) stand for, in 32 bits."""
    t = q.float().reshape(q.shape[0], -1, BLOCK)
    return (t * _power(byte[:, :t.shape[1], None])).reshape(q.shape)


def _rounded(x, rows):
    return _values(*_quantized(x, rows))


def _linear_plain(s):
    case = s["case"]
    out = TYPES[case["out"]]
    w = _values(*s["weight8"]) if "weight8" in s else _rounded(s["weight"], BLOCK)
    y = _rounded(s["x"], 1) @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["form"] != "train":
        return y.to(out)
    n, k = case["n"], case["k"]
    dy, x = s["dy"], s["x"]
    wt = _rounded(s["weight"].t(), BLOCK)
    dx = (_rounded(dy, 1) @ wt.t())[:, :k]
    dw = _rounded(dy.t(), 1) @ _rounded(x.t(), 1).t()
    grads = {"y": y[:, :n].to(out), "dx": dx.to(x.dtype), "dw": dw.to(s["weight"].dtype)}
    if s["bias"] is not None:
        grads["db"] = dy.float().sum(0)
    return grads


def _distill_plain(s):
    case = s["case"]
    t, v = case["t"], case["v"]
    z = s["student"].float() / t
    z = z - z.amax(dim=1, keepdim=True)
    e = z.exp()
    total = e.sum(dim=1, keepdim=True)
    good = (s["index"] >= 0) & (s["index"] < v)
    at = torch.where(good, s["index"], 0).long()
    a = torch.where(good, s["teacher"].float() / t, float("-inf"))
    a = a - a.amax(dim=1, keepdim=True)
    some = good.any(dim=1, keepdim=True)
    a = torch.where(some, a, 0.0)
    p = torch.where(good, a.exp(), 0.0)
    share = p.sum(dim=1, keepdim=True)
    share = torch.where(some, share, 1.0)
    p = p / share
    logq = torch.gather(z, 1, at) - total.log()
    loss = torch.where(p > 0, p * (a - share.log() - logq), 0.0).sum(dim=1)
    if case["form"] == "loss":
        return loss
    scale = (s["upstream"] / t)[:, None] * some
    dz = (e / total) * scale
    dz.scatter_add_(1, at, -p * scale)
    return {"loss": loss, "grad": dz.to(s["student"].dtype)}


def _column(x, like):
    """A setting for every row: a number, or one a row."""
    return x.to(like.dtype)[:, None] if isinstance(x, torch.Tensor) else torch.full((like.shape[0], 1), float(x), dtype=like.dtype, device=like.device)


def _draw_plain(s):
    z = s["logits"].double()            # values next to a border: 64 bits
    t, top_k, top_p, min_p = (_column(s[q], z) for q in ("t", "top_k", "top_p", "min_p"))
    order, at = torch.sort(z, dim=1, descending=True, stable=True)
    some = order[:, :1] > float("-inf")
    p = torch.where(order > float("-inf"), ((order - order[:, :1]) / t).exp(), 0.0)
    place = torch.arange(z.shape[1], device=z.device)
    p = torch.where((top_k <= 0) | (place < top_k), p, 0.0)
    before = p.cumsum(dim=1) - p
    p = torch.where((top_p >= 1) | (before < top_p * p.sum(dim=1, keepdim=True)) | (place == 0), p, 0.0)
    p = torch.where(p >= min_p, p, 0.0)
    running = p.cumsum(dim=1)
    place = (running <= s["u"].double()[:, None] * running[:, -1:]).sum(dim=1, keepdim=True)
    last = (running < running[:, -1:]).sum(dim=1, keepdim=True)
    return torch.where(some, at.gather(1, torch.minimum(place, last)), -1)[:, 0]


def run(state):
    if own:
        return _run_own(state)
    return {"linear": _linear_plain, "distill": _distill_plain, "draw": _draw_plain}[state["case"]["op"]](state)


# ---- the framework's calls -----------------------------------------------------------------------------------------------

def _run_own(s):
    import object_nerf_amd as A
    case = s["case"]
    if case["op"] == "draw":
        return A.sample_logits(s["logits"], s["u"], temperature=s["t"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    if case["op"] == "distill":
        if case["form"] == "loss":
            return A.distill_top_logits(s["student"], s["teacher"], s["index"], temperature=case["t"])
        if case["form"] == "grad":
            loss, grad = A.distill_top_logits_grad(s["student"], s["teacher"], s["index"], s["upstream"], temperature=case["t"])
            return {"loss": loss, "grad": grad}
        z = s["student"].detach().requires_grad_()
        loss = A.distill_top_logits(z, s["teacher"], s["index"], temperature=case["t"])
        return {"loss": loss.detach(), "grad": torch.autograd.grad(loss, z, s["upstream"])[0]}
    out = TYPES[case["out"]]
    if case["form"] != "train":
        return A.linear_fp8(s["x"], A.Fp8Matrix(*s["weight8"], case["k"]), s["bias"], out_dtype=out)
    x, w = s["x"].detach().requires_grad_(), s["weight"].detach().requires_grad_()
    b = None if s["bias"] is None else s["bias"].detach().requires_grad_()
    y = A.linear_fp8(x, w, b, out_dtype=out)
    got = torch.autograd.grad(y, [x, w] + ([] if b is None else [b]), s["dy"])
    return dict(zip(("y", "dx", "dw", "db"), (y.detach(),) + got))


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def _exact_e4m3(x, rows):
    """x (R, C) in 64 bits, every value replaced by the nearest one of its block's grid (ties to even): 3 bits behind the
    leading one, no exponent under -6, times the block's power of two."""
    x = x.double()
    r, c = x.shape
    padded = torch.zeros(-(-r // rows) * rows, -(-c // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    padded[:r, :c] = x
    largest = padded.abs().reshape(padded.shape[0], -1, BLOCK).amax(2)
    largest = largest.reshape(-1, rows, largest.shape[1]).amax(1).repeat_interleave(rows, 0).repeat_interleave(BLOCK, 1)
    scale = torch.exp2(torch.ceil(torch.log2(torch.clamp(largest, min=1e-300) / 448.0)).clamp(min=-126))
    scale = torch.where(largest > scale * 448.0, scale * 2, torch.where((largest * 2 <= scale * 448.0) & (scale > 2.0 ** -126), scale / 2, scale))
    u = padded / scale
    grid = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(u / grid) * grid * scale)[:r, :c]


def _exact_linear(s, case):
    x = _exact_e4m3(s["x"], 1)
    if case["form"] == "train":
        w = _exact_e4m3(s["weight"], BLOCK)
    else:
        q, byte = s["weight8"]
        w = (q.double() * torch.exp2(byte.double() - 127).repeat_interleave(BLOCK, 1)[:, :q.shape[1]])[:, :case["k"]]
    y = torch.mm(x, w.t().contiguous())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["form"] != "train":
        return y
    dy = s["dy"].double()
    got = {"y": y, "dx": torch.mm(_exact_e4m3(dy, 1), w), "dw": torch.mm(_exact_e4m3(dy.t(), 1), _exact_e4m3(s["x"].double().t(), 1).t().contiguous())}
    if s["bias"] is not None:
        got["db"] = dy.sum(0)
    return got


def _exact_distill(s, case):
    v, t = case["v"], case["t"]
    ok = (s["index"] >= 0) & (s["index"] < v)
    slot = s["index"].long().clamp(0, v - 1)
    dead = ~ok.any(1)
    logq = s["student"].double() / t
    logq = logq - torch.logsumexp(logq, 1, keepdim=True)
    a = (s["teacher"].double() / t).masked_fill(~ok, float("-inf"))
    a[dead] = 0.0
    logp = a - torch.logsumexp(a, 1, keepdim=True)
    p = logp.exp() * ok
    p[dead] = 0.0
    loss = (p * (torch.where(p > 0, logp, 0.0) - logq.gather(1, slot))).sum(1)
    if case["form"] == "loss":
        return loss
    target = torch.zeros_like(logq).scatter_add_(1, slot, p)
    grad = (logq.exp() * p.sum(1, keepdim=True) - target) * (s["upstream"].double() / t)[:, None]
    return {"loss": loss, "grad": grad}


def _exact_draw(s, case):
    """Over blocks of rows, by every label's rank: a label is kept if it comes before the cut in (value, index) order."""
    z = s["logits"].double()
    out = []
    setting = {q: _column(s[q], z) for q in ("t", "top_k", "top_p", "min_p")}
    for at in range(0, z.shape[0], 4096):
        rows = slice(at, at + 4096)
        zz, t, k, tp, mp = z[rows], *(setting[q][rows] for q in ("t", "top_k", "top_p", "min_p"))
        weight = torch.exp((zz - zz.amax(1, keepdim=True).clamp(min=-1e308)) / t)
        rank = torch.argsort(torch.argsort(-zz, dim=1, stable=True), dim=1)
        weight = weight * ((k <= 0) | (rank < k))
        ranked = torch.zeros_like(weight).scatter_(1, rank, weight)
        share = torch.zeros_like(weight)
        share[:, 1:] = ranked.cumsum(1)[:, :-1]
        kept = (share.gather(1, rank) < tp * weight.sum(1, keepdim=True)) | (rank == 0) | (tp >= 1)
        weight = weight * kept * (weight >= mp)
        running = torch.zeros_like(weight).scatter_(1, rank, weight).cumsum(1)
        target = s["u"][rows].double()[:, None] * running[:, -1:]
        place = torch.searchsorted(running, target, right=True)
        out.append(torch.where(running[:, -1] > 0, (rank == place).to(torch.uint8).argmax(1), -1))
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "distill": _exact_distill, "draw": _exact_draw}[case["op"]](s, case)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def _bytes(kind):
    return 4 if kind == "fp32" else 2


def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        e = _bytes(case["type"])
        if case["form"] == "train":     # x, w and dy in; y, dx and dw out
            return {"bytes": 2 * e * (m * k + n * k + m * n) + (8 * n if case["bias"] else 0), "flops": 6 * m * n * k}
        return {"bytes": e * m * k + n * k + _bytes(case["out"]) * m * n + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    n, v = case["n"], case["v"]
    if case["op"] == "distill":
        top = n * case["k"] * (_bytes(case["teacher"]) + 4) + 4 * n
        if case["form"] == "loss":
            return {"bytes": n * v * _bytes(case["type"]) + top, "flops": 3 * n * v}
        return {"bytes": 2 * n * v * _bytes(case["type"]) + top + 4 * n, "flops": 6 * n * v}
    return {"bytes": n * v * _bytes(case["type"]) + n * (4 + 8) + (16 * n if case["rows"] else 0), "flops": 3 * n * v}
