"""Plain 64-bit forms of the label operators on the CPU, for the tests: formulas, one row or one matrix at a time."""
import math

import torch

STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step, relative


def distill(student, teacher, index, upstream, temperature):
    """(loss, grad, size) in float64; size: the two terms of the gradient added instead of subtracted, (upstream / T) (q + p)"""
    z, t, idx = student.detach().cpu().double(), teacher.detach().cpu().double(), index.cpu().long()
    n, v = z.shape
    loss, grad, size = (torch.zeros(s, dtype=torch.float64) for s in ((n,), (n, v), (n, v)))
    for r in range(n):
        slots = [j for j in range(idx.shape[1]) if 0 <= idx[r, j] < v and t[r, j] != -math.inf]
        if not slots:
            continue
        at, x = idx[r, slots], t[r, slots] / temperature
        logp = x - torch.logsumexp(x, 0)
        logq = z[r] / temperature - torch.logsumexp(z[r] / temperature, 0)
        p = logp.exp()
        loss[r] = torch.where(p > 0, p * (logp - logq[at]), torch.zeros_like(p)).sum()
        target = torch.zeros(v, dtype=torch.float64).index_add_(0, at, p)
        grad[r] = (logq.exp() - target) * (float(upstream[r]) / temperature)
        size[r] = (logq.exp() + target) * (float(upstream[r]) / temperature)
    return loss, grad, size


def order_of(z):
    """the labels of one row in order: falling logit, equal ones by rising index, without -inf / NaN"""
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z.double())
    order = torch.sort(z, descending=True, stable=True)[1]
    return order[z[order] > -math.inf], z


def sample(logits, u, temperature, top_k, top_p, min_p):
    """labels by the definition, row by row (settings: numbers or per-row lists)"""
    n = logits.shape[0]
    per_row = lambda s: [float(x) for x in s] if isinstance(s, torch.Tensor) else [float(s)] * n       # noqa: E731
    out = []
    for r, (t, k, tp, mp, uu) in enumerate(zip(per_row(temperature), per_row(top_k), per_row(top_p), per_row(min_p), per_row(u))):
        order, z = order_of(logits[r].cpu())
        if not len(order):
            out.append(-1)
            continue
        if not t > 0:
            out.append(int(order[0]))
            continue
        x = z[order]
        w = torch.where(x == x[0], torch.ones_like(x), torch.exp((x - x[0]) / t))
        if k >= 1:
            w = w[:int(k)]
        if tp < 1:
            before = torch.cumsum(w, 0) - w
            before[0] = -1.0
            w = w[before < tp * w.sum()]
        w = w[w >= min(mp, 1.0)]
        run = torch.cumsum(w, 0)
        place = int((run <= min(max(uu, 0.0), 1.0) * run[-1]).sum())
        last = int((run < run[-1]).sum())
        out.append(int(order[min(place, last)]))
    return torch.tensor(out)


def fp8(x, block_rows):
    """the values that x (R, C) stands for in e4m3 with a power-of-two scale per block of block_rows x 128, in float64, and the scale
    bytes (R, blocks)"""
    x = x.detach().cpu().double()
    r, c = x.shape
    out, scale = torch.zeros_like(x), torch.zeros(r, -(-c // 128), dtype=torch.int64)
    for b in range(scale.shape[1]):
        for top in range(0, r, block_rows):
            blk = x[top:top + block_rows, b * 128:(b + 1) * 128]
            mag = torch.where(torch.isfinite(blk), blk.abs(), torch.zeros_like(blk))
            largest = float(mag.max())
            e = 0
            if largest > 0:
                e = math.frexp(largest)[1] - 10
                while largest > 448.0 * 2.0 ** e:
                    e += 1
                e = max(e, -126)
            u = blk / 2.0 ** e
            grid = 2.0 ** (torch.clamp(torch.frexp(u)[1] - 1, min=-6).double() - 3)
            out[top:top + block_rows, b * 128:(b + 1) * 128] = torch.where(torch.isfinite(u), torch.round(u / grid) * grid * 2.0 ** e, torch.full_like(u, math.nan))
            scale[top:top + block_rows, b] = 127 + e
    return out, scale
