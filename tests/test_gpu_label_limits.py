"""GPU: the label operators at the ends of what they take."""
import math

import pytest
import torch

import label_reference as R
import object_nerf_amd as A

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- drawing a label ----

@pytest.mark.parametrize("weak", [-14.0, -20.0, -28.0, -30.0])
def test_sample_one_strong_label_over_the_flattest_and_longest_tail(weak):
    """Weights are whole numbers of 2^-43 at 2^19 labels: each is off by 2^-44 at most, a sum of them by 2^-25 of the strong one.  u times the
    total lies between the running sums in front of and behind the label, off by that twice."""
    v, strong = 1 << 19, 12345
    z = torch.full((1, v), weak, device=DEV)
    z[0, strong] = 0.0
    u = torch.tensor([0.0, 0.5, 1 - 2.0 ** -6, 1 - 2.0 ** -12, 1 - 2.0 ** -18, 1 - 2.0 ** -22, 1 - 2.0 ** -24])
    w = math.exp(weak)
    total = 1 + (v - 1) * w
    for rows in (1, len(u)):                                    # a row over several workgroups; rows at a time
        for at in range(0, len(u), rows):
            labels = A.sample_logits(z.expand(rows, v), u[at:at + rows].to(DEV)).tolist()
            for label, x in zip(labels, u[at:at + rows].tolist()):
                rank = 0 if label == strong else label + (label < strong)
                front, behind = (0.0, 1.0) if rank == 0 else (1 + (rank - 1) * w, 1 + rank * w)
                assert front - 2.0 ** -24 <= x * total <= behind + 2.0 ** -24, (x, label)


def test_sample_refuses_longer_rows():
    with pytest.raises(ValueError, match="2\\^19"):
        A.sample_logits(torch.zeros(1, (1 << 19) + 1, device=DEV), torch.zeros(1, device=DEV))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.uint16, torch.uint32, torch.int64, torch.uint64])
def test_sample_top_k_per_row_of_any_whole_type(dtype):
    n, v = 12, 700
    g = _gen(8)
    z, u = torch.randn(n, v, generator=g), torch.rand(n, generator=g)
    most = torch.iinfo(dtype).max
    k = [0, 1, 5, 100, min(most, 650), most, most // 2 + 1, min(most, 1 << 31), min(most, (1 << 32) - 1), min(most, (1 << 32) + 3), min(most, 1 << 62), 7]
    label = A.sample_logits(z.to(DEV), u.to(DEV), top_k=torch.tensor(k, dtype=dtype).to(DEV))
    assert torch.equal(label.cpu(), R.sample(z, u, 1.0, torch.tensor([min(x, v) for x in k]), 1.0, 0.0))


def test_labels_of_rays_with_an_infinite_feature_go_into_the_table():
    """as the documentation has it: -1 clamped for the lookup, and known"""
    g = _gen(2)
    features, weight = torch.randn(30, 40, generator=g), torch.randn(64, 40, generator=g)
    features[7, 3], features[11, 0] = math.inf, math.nan
    ids = A.sample_logits(A.linear_fp8(features.to(DEV), A.quantize_fp8(weight.to(DEV), block_rows=128)), torch.rand(30, generator=g).to(DEV), temperature=0.8, top_k=8)
    known = ids >= 0
    assert (~known).nonzero().flatten().tolist() == [7, 11]
    codes = A.CodeLibrary(A.default_model_config()).to(DEV)
    code = codes({"instance_ids": ids.clamp(min=0)})["embedding_instance"]
    assert torch.equal(code.detach()[known], codes.embedding_instance.weight.detach()[ids[known]])


# ---- views that stand for minus their memory ----

@pytest.mark.parametrize("v", [1, 40])
def test_negated_views(v):
    g = _gen(v)
    c = torch.complex(torch.randn(6, v, generator=g), torch.randn(6, v, generator=g)).to(DEV)
    u, t, i = torch.rand(6, generator=g).to(DEV), torch.randn(6, 2, generator=g).to(DEV), torch.randint(0, v, (6, 2), generator=g).to(DEV)
    for view in (c.conj().imag, torch._neg_view(c.real.contiguous())):
        assert view.is_neg()
        plain = view.resolve_neg().contiguous()
        assert torch.equal(A.sample_logits(view, u), A.sample_logits(plain, u))
        assert torch.equal(A.linear_fp8(view, view, view[:, 0]), A.linear_fp8(plain, plain, plain[:, 0]))
        assert torch.equal(A.quantize_fp8(view).data.view(torch.uint8), A.quantize_fp8(plain).data.view(torch.uint8))
        for got, want in zip(A.distill_top_logits_grad(view, t, i, view[:, 0]), A.distill_top_logits_grad(plain, t, i, plain[:, 0])):
            assert torch.equal(got, want)
        assert torch.equal(A.distill_top_logits(plain, torch._neg_view(t), i), A.distill_top_logits(plain, -t, i))
        leaf = plain.requires_grad_()
        for out in (A.distill_top_logits(leaf, t, i), A.linear_fp8(leaf, leaf.detach())):
            d = torch.randn(out.shape, generator=g).to(DEV)
            assert torch.equal(*(torch.autograd.grad(out, leaf, x, retain_graph=True)[0] for x in (torch._neg_view(d), -d)))


# ---- distillation ----

def test_distill_refuses_more_labels_than_its_sizes_hold():
    """2^32 + 5 labels would be 5 in 32 bits"""
    one = torch.zeros(1, 1, device=DEV)
    z = torch.empty(1, (1 << 32) + 5, dtype=BF16, device=DEV)                   # refused before anything reads it
    for call in (lambda: A.distill_top_logits(z, one, one.long()), lambda: A.distill_top_logits_grad(z, one, one.long(), one[0]),
                 lambda: A.distill_top_logits(z.requires_grad_(), one, one.long())):
        with pytest.raises(ValueError, match="2\\^31"):
            call()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v,k", [(40, 4), (40, 30), (900, 4), (5000, 70), (70001, 4)])
def test_distill_lowest_values_under_slots(v, k, dtype):
    """Masked labels under filled slots: the terms, up to 2^129, are brought back by their weights, their mean or T.  Relative error of a
    loss: exp at distances up to 80 with three roundings of the argument, the term and the sums of k of them; all terms have one sign,
    next to which the logarithms are nothing."""
    low = torch.finfo(dtype).min
    z, t, i = torch.zeros(7, v), torch.full((7, k), -math.inf), torch.arange(k).expand(7, k).clone()
    t[:, :4] = torch.tensor([0.5, 0.25, 0.0, -1.0])
    z[0, 0] = low                                         # one of four
    z[1, :4] = low                                        # every slot: the terms' sum is over fp32's end
    z[2, 0], t[2, 0] = low, -70.0                         # next to no weight
    z[3, 3], t[3, 3] = low, -30.0
    z[4], t[4, 1:] = low, -math.inf                       # the whole row masked: alike
    z[5, 2], z[5, 7] = low, -low                          # the whole range of the type
    z[6, 1], t[6, 1], i[6, 2] = low, -20.0, 1             # an index twice
    u = torch.full((7,), 0.125)
    z = z.to(dtype)
    for temperature in (0.25, 0.5, 1.0, 3.0):
        loss, grad = A.distill_top_logits_grad(z.to(DEV), t.to(DEV), i.to(DEV), u.to(DEV), temperature=temperature)
        # (rows less their largest: 64 bits would lose log v next to 1e39, and a softmax does not see the shift)
        rl, rg, _ = R.distill(z.double() - z.double().amax(1, keepdim=True), t, i, u, temperature)
        held = rl.abs() < torch.finfo(F32).max * (1 - 2.0 ** -12)               # else: an infinity, or next to one
        assert held[2:5].all() and torch.equal(torch.isinf(loss.cpu())[held], torch.zeros(int(held.sum()), dtype=torch.bool))
        assert (loss.cpu()[~held] >= torch.finfo(F32).max * (1 - 2.0 ** -11)).all()
        d = 80 / min(temperature, 1.0)
        bound = (3 * d + k + 20) * R.STEP[F32] * rl.abs() + (80 + v / 256 + k) * R.STEP[F32] * (1 + math.log(v))
        assert ((loss.cpu().double() - rl).abs()[held] <= bound[held]).all(), ((loss.cpu().double() - rl) / bound)
        assert torch.equal(A.distill_top_logits(z.to(DEV), t.to(DEV), i.to(DEV), temperature=temperature), loss)
        size = (3 * d + v / 256 + k + 20) * R.STEP[F32] * 0.25 / temperature
        assert ((grad.cpu().double() - rg).abs() <= R.STEP[dtype] * rg.abs() + size + (2.0 ** -24 if dtype == F16 else 0)).all()


@pytest.mark.parametrize("v,k", [(40, 2), (3000, 70), (70001, 2)])
def test_distill_ruled_out_labels_cost_infinity_at_any_weight(v, k):
    z, t, i = torch.zeros(3, v), torch.full((3, k), -math.inf), torch.arange(k).expand(3, k)
    z[:, 0] = -math.inf
    t[:, 0], t[:, 1] = torch.tensor([0.0, -90.0, -1e30]), 0.0                   # weights of 1/2 and less than fp32 holds
    loss, grad = A.distill_top_logits_grad(z.to(DEV), t.to(DEV), i.to(DEV), torch.ones(3, device=DEV))
    assert (loss == math.inf).all() and torch.isfinite(grad).all()
    t[:, 0] = -math.inf                                                         # an empty slot costs nothing
    assert torch.isfinite(A.distill_top_logits(z.to(DEV), t.to(DEV), i.to(DEV))).all()


# ---- products in 8-bit floating point ----

def _values(q):
    return (q.data.double() * torch.exp2(q.scale.double() - 127).repeat_interleave(128, 1)[:, :q.data.shape[1]])[:, :q.cols]


@pytest.mark.parametrize("m,n,k,dtype", [(5, 300, 130, F32), (30, 70, 4000, BF16), (200, 100, 300, F32), (200, 100, 300, BF16), (130, 520, 9000, F32), (70000, 70, 200, BF16), (300, 1000, 128, F32)])
def test_linear_fp8_smallest_scales(m, n, k, dtype):
    """Blocks whose values reach down to where bf16, through which fp32 results go, has no more bits.  Scales of 2^-126 and 2^-125 in some rows
    of either factor and in some blocks of a row, next to scales that bring the results back; 64-bit sums with the bound of fp32 ones:
    two roundings a term, of the sum of magnitudes, where fp32 holds that sum."""
    g = _gen(m + n)
    x, w = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g)
    x[::3] *= 2.0 ** torch.randint(-131, -110, (len(x[::3]), 1), generator=g)
    x[1::3, :100] *= 2.0 ** -120
    w[:128] *= 2.0 ** 90
    w[128:256] *= 2.0 ** -124
    x[2::3] *= 2.0 ** 30
    x = x.to(dtype)
    q, w8 = A.quantize_fp8(x.to(DEV)), A.quantize_fp8(w.to(DEV), 128)
    assert (q.scale < 3).any() and (n <= 128 or (w8.scale < 3).any())
    a, b = _values(q), _values(w8)
    want, size = a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    bound = torch.where(size < 2.0 ** 127, (k + 2) * 2 * R.STEP[F32] * size + 2.0 ** -126, math.inf)
    assert (bound < math.inf).double().mean() > 0.5
    for y in (A.linear_fp8(x.to(DEV), w8, out_dtype=F32), A.matmul_fp8(q, w8, out_dtype=F32)):
        far = ((y.double() - want).abs() > bound) & (bound < math.inf)
        assert not far.any(), ((y.double() - want).abs() / bound)[far].max().item()
    rows = A.matmul_fp8(q, w8, out_dtype=F32)[1]
    other = A.quantize_fp8(torch.cat([x[1:2], torch.randn(40, k, generator=g).to(dtype)]).to(DEV))          # rows do not see their neighbours' scales
    assert not (((A.matmul_fp8(other, w8, out_dtype=F32)[0].double() - rows.double()).abs() > bound[1]) & (bound[1] < math.inf)).any()


PRODUCTS = [(5, 300, 130), (16, 4096, 1000), (30, 70, 4000), (64, 64, 8000), (200, 100, 300), (389, 520, 9000), (1000, 96, 256), (4000, 3700, 1100), (70000, 70, 200), (9000, 1100, 130)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("out", [F32, BF16, F16])
def test_linear_fp8_counts_every_product_once(m, n, k, out):
    """Whole numbers whose sums every type holds, under scales that differ from row to row and block to block: nothing is rounded or dropped,
    so a lost, doubled or wrongly scaled product shows.  Rows of x: +-1 at twelve places; weights: whole numbers up to 7."""
    g = torch.Generator(device=DEV).manual_seed(m + k)
    kb, nb = -(-k // 128), -(-n // 128)
    x = torch.zeros(m, k, device=DEV)
    at = torch.randint(0, k, (m, 12), device=DEV, generator=g)
    x.scatter_(1, at, torch.where(torch.rand(m, 12, device=DEV, generator=g) < 0.5, -1.0, 1.0))
    w = torch.randint(-7, 8, (n, k), device=DEV, generator=g).float()
    want = torch.mm(x, w.t().contiguous())                                      # whole numbers up to 84: exact in fp32 in any order
    p = torch.exp2(torch.randint(-20, 21, (kb,), device=DEV, generator=g).float()).repeat_interleave(128)[:k]
    r = torch.exp2(torch.randint(-3, 4, (m, 1), device=DEV, generator=g).float())
    c = torch.exp2(torch.randint(-2, 3, (nb,), device=DEV, generator=g).float()).repeat_interleave(128)[:n]
    want = want * r * c
    w8 = A.quantize_fp8(w / p * c[:, None], 128)
    for y in (A.linear_fp8(x * p * r, w8, out_dtype=out), A.matmul_fp8(A.quantize_fp8(x * p * r), w8, out_dtype=out)):
        assert torch.equal(y.float(), want)


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("out", [BF16, F16])
def test_matmul_fp8_precision_of_16_bit_results(m, n, k, out):
    """The instruction's error d before the rounding is 1.5e-5 of the result's norm (measured); 3e-5 is let through.  round(x + d) and
    round(x) differ by whole steps of at most 2 h |x| (h: half a step), by |d| on average, so their squared distance is 2 h |x| |d| on
    average and in norm at most sqrt(2 h 3e-5) of x; a tenth more for the average being one of a sample."""
    g = torch.Generator(device=DEV).manual_seed(n)
    a, b = A.quantize_fp8(torch.randn(m, k, device=DEV, generator=g)), A.quantize_fp8(torch.randn(n, k, device=DEV, generator=g), 128)
    want = torch.mm(_values(a), _values(b).t().contiguous())
    for y in (A.matmul_fp8(a, b, out_dtype=out), A.linear_fp8(_values(a).to(BF16), b, out_dtype=out)):        # 4 bits: x again what it was
        off = (y.double() - want.to(out).double()).norm() / want.norm()
        assert off.item() <= 1.1 * (2 * R.STEP[out] * 3e-5) ** 0.5


def test_results_and_rows_past_32_bits():
    """more than 2^31 results, 2^32 bytes of 8-bit values and of logits: the rows around those ends against the same rows by themselves"""
    g = torch.Generator(device=DEV).manual_seed(1)
    m, n, k = 600000, 8000, 130
    x, w8 = torch.randn(m, k, device=DEV, generator=g).to(BF16), A.quantize_fp8(torch.randn(n, k, device=DEV, generator=g), 128)
    ends = [0, (1 << 31) // n, (1 << 32) // n, m - 1]
    for y in (A.linear_fp8(x, w8), A.matmul_fp8(A.quantize_fp8(x), w8)):
        for at in ends:
            rows = slice(max(0, at - 20), at + 20)
            assert torch.equal(y[rows], A.linear_fp8(x[rows], w8)) or (y[rows].double() - A.linear_fp8(x[rows], w8).double()).norm() <= 1e-3 * y[rows].double().norm()
        u, t, i = torch.rand(m, device=DEV, generator=g), torch.randn(m, 3, device=DEV, generator=g), torch.randint(0, n, (m, 3), device=DEV, generator=g)
        label, (loss, grad) = A.sample_logits(y, u, top_p=0.9), A.distill_top_logits_grad(y, t, i, u)
        for at in ends:
            rows = slice(max(0, at - 20), at + 20)
            assert torch.equal(label[rows], A.sample_logits(y[rows], u[rows], top_p=0.9))
            for got, want in zip((loss, grad), A.distill_top_logits_grad(y[rows], t[rows], i[rows], u[rows])):
                assert torch.equal(got[rows], want)
        del label, loss, grad
    for block_rows in (1, 128):
        for transpose in (False, True):
            q = A.quantize_fp8(y, block_rows, transpose)
            for at in ((1 << 31) // n, (1 << 32) // n, m - 130):
                at -= at % 128
                want = A.quantize_fp8(y[at:at + 128], block_rows, transpose)
                data, scale = (q.data[:, at:at + 128], q.scale[:, at // 128:at // 128 + 1]) if transpose else (q.data[at:at + 128], q.scale[at:at + 128])
                assert torch.equal(data.view(torch.uint8), want.data.view(torch.uint8)) and torch.equal(scale, want.scale[:, :scale.shape[1]])
            del q


# ---- derivatives ----

def test_forward_mode_over_backward_is_refused():
    fw = torch.autograd.forward_ad
    x, w = torch.randn(4, 6, device=DEV, requires_grad=True), torch.randn(5, 6, device=DEV)
    z, t, i = torch.randn(4, 6, device=DEV, requires_grad=True), torch.randn(4, 2, device=DEV), torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    y, loss = A.linear_fp8(x, w), A.distill_top_logits(z, t, i)
    with fw.dual_level():
        for out, leaf in ((y, x), (loss, z)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaf, fw.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            q = A.quantize_fp8(w)
            A.matmul_fp8(q, q, fw.make_dual(torch.ones(5, device=DEV), torch.ones(5, device=DEV)))
        label = A.sample_logits(fw.make_dual(z.detach(), torch.ones_like(z)), torch.rand(4, device=DEV))      # whole numbers have no derivative
        assert label.shape == (4,)
    assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape


# ---- torch.compile: the calls stay as they are, between compiled parts ----

def test_calls_inside_a_compiled_function():
    g = _gen(3)
    x, w, b = (torch.randn(*s, generator=g).to(DEV).requires_grad_() for s in ((7, 40), (12, 40), (12,)))
    t, i, u = torch.randn(7, 3, generator=g).to(DEV), torch.randint(-1, 12, (7, 3), generator=g).to(DEV), torch.rand(7, generator=g).to(DEV)

    def step(x, w, b):
        y = A.linear_fp8(x * 2, w, b)
        loss = A.distill_top_logits(y, t, i)
        both = A.distill_top_logits_grad(y.detach(), t, i, u)
        label = A.sample_logits(y.detach(), u, top_k=3)
        return (loss * 2).sum(), both[0] + 1, both[1] * 2, label + 1

    got, want = torch.compile(step, backend="eager")(x, w, b), step(x, w, b)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    for p, q in zip(torch.autograd.grad(got[0], (x, w, b)), torch.autograd.grad(want[0], (x, w, b))):
        assert torch.equal(p, q)
