"""GPU: the operators of a training step (deepsignal_plant_amd/train_ops.py) against plain implementations in 64 bits, at the
sizes, types and values where they can go wrong.  A rounding to a type is off by at most finfo(type).eps / 2 of the value (and
by half of the smallest subnormal); the sums' bounds stand at each check."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24   # half a step of float32, relative
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from deepsignal_plant_amd import train_ops
    return train_ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rounding(want, dtype):
    """largest error of rounding `want` (float64) to dtype once"""
    return want.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def close(got, want, bound, what=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), what
    off = (got - want).abs()
    off[nan | (got == want)] = 0
    bad = off > bound.masked_fill(nan, math.inf) if isinstance(bound, torch.Tensor) else off > bound
    assert not bad.any(), "%s: %d of %d off, the worst by %g" % (what, int(bad.sum()), bad.numel(), float(off[bad].max()))


# ---- embedding -------------------------------------------------------------------------------------------------------------------
def check_embedding(ops, tokens, weight, scale=1.0, padding_idx=None, seed=3):
    """weight, tokens on the GPU.  The forward is one product in 32 bits, rounded; a row's gradient a sum of k products, each
    addition off by at most U of the partial sum: at most k U sum |g| |scale|, the scale's rounding and the type's on top"""
    w = weight.detach().requires_grad_()
    out = ops.embedding(tokens, w, scale=scale, padding_idx=padding_idx)
    t = tokens.cpu().to(torch.int64).reshape(-1)
    rows, dim = weight.shape
    bad = (t < 0) | (t >= rows)
    s = float(np.float32(scale))
    wd = weight.detach().cpu().double()
    want = wd[t.clamp(0, rows - 1)] * s
    want[bad] = math.nan
    want = want.view(*tokens.shape, dim)
    close(out, want, rounding(want, weight.dtype) + U * want.abs(), "forward")
    assert out.dtype == weight.dtype
    g = torch.randn(*tokens.shape, dim, generator=gen(seed)).to(weight.dtype)
    dw, = torch.autograd.grad(out, w, g.to(weight.device))
    assert dw.dtype == weight.dtype
    gd = g.double().reshape(-1, dim)
    use = ~bad if padding_idx is None else ~bad & (t != padding_idx % rows)
    total, size, count = torch.zeros(rows, dim, dtype=torch.float64), torch.zeros(rows, dim, dtype=torch.float64), torch.zeros(rows, 1, dtype=torch.float64)
    total.index_add_(0, t[use], gd[use])
    size.index_add_(0, t[use], gd[use].abs())
    count.index_add_(0, t[use], torch.ones(int(use.sum()), 1, dtype=torch.float64))
    want = total * s
    close(dw, want, (count + 1) * U * size * abs(s) + rounding(want, weight.dtype), "gradient")
    again, = torch.autograd.grad(ops.embedding(tokens, w, scale=scale, padding_idx=padding_idx), w, g.to(weight.device))
    assert torch.equal(again, dw)   # whatever the order of arrival


def tokens_of(n, rows, dtype=torch.int64, seed=1):
    return torch.randint(0, rows, (n,), generator=gen(seed)).to(dtype).to(DEV)


def table(rows, dim, dtype=F32, seed=2):
    return torch.randn(rows, dim, generator=gen(seed)).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [1, 2, 3, 4, 7, 8, 64, 100, 257, 1024])
def test_embedding_rows_of_every_width(ops, dim, dtype):
    for rows, n in ((16, 333), (900, 1500)):
        check_embedding(ops, tokens_of(n, rows), table(rows, dim, dtype), scale=1.7)


@pytest.mark.parametrize("n", [0, 1, 2, 3, 63, 64, 65, 255, 257, 1023, 1024, 1025, 4095, 4096, 4097, 8192, 8193, 70001])
@pytest.mark.parametrize("rows", [1, 2, 16, 64, 65, 1000, 1023, 1024, 70000])
def test_embedding_lengths_and_tables(ops, n, rows):
    check_embedding(ops, tokens_of(n, rows, torch.int32), table(rows, 4))


@pytest.mark.parametrize("rows,dim,n", [(16, 4, 852000), (64, 4, 200000), (63, 3, 150001), (60, 256, 40000), (256, 1, 140000), (300, 64, 60000)])
def test_embedding_many_tokens_of_small_tables(ops, rows, dim, n):
    check_embedding(ops, tokens_of(n, rows, torch.int32), table(rows, dim))
    check_embedding(ops, tokens_of(n, rows, torch.int32), table(rows, dim, BF16), scale=3.0)


@pytest.mark.parametrize("rows,dim", [(16, 4), (5000, 24), (300000, 8), (2 ** 21, 1)])
def test_embedding_one_token_takes_all(ops, rows, dim):
    """a run over every chunk of the sorted order, and all but a few"""
    t = torch.full((9000,), rows - 1, dtype=torch.int64)
    check_embedding(ops, t.to(DEV), table(rows, dim))
    t[::700] = 0
    t[1::900] = rows // 2
    check_embedding(ops, t.to(DEV), table(rows, dim, BF16), scale=0.5)


@pytest.mark.parametrize("runs", [(15, 16, 17), (16, 16, 16), (1, 62, 1, 64, 129), (63, 65, 128, 1), (200, 1, 1, 1, 300)])
@pytest.mark.parametrize("copies", [1, 120])
def test_embedding_runs_that_end_at_and_around_the_chunks(ops, runs, copies):
    t = torch.cat([torch.full((k,), 7 * i) for i, k in enumerate(runs * copies)])
    check_embedding(ops, t[torch.randperm(len(t), generator=gen(9))].to(DEV), table(7 * len(runs) * copies + 1, 20))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.uint16, torch.int32, torch.int64, F32])
@pytest.mark.parametrize("rows", [16, 200])
def test_embedding_token_types(ops, dtype, rows):
    check_embedding(ops, tokens_of(13 * 40, rows).to(dtype).view(40, 13), table(rows, 12))


@pytest.mark.parametrize("rows", [16, 700])
def test_embedding_tokens_outside_the_table(ops, rows):
    """a row of NaN, and no gradient; nothing beside it is touched"""
    t = tokens_of(500, rows)
    t[3], t[100], t[499], t[77] = -1, rows, 2 ** 40, -2 ** 40
    check_embedding(ops, t, table(rows, 8))
    f = t.float()
    f[5], f[6], f[7] = math.nan, math.inf, -math.inf
    w = table(rows, 8).requires_grad_()
    out = ops.embedding(f, w)
    assert torch.isnan(out[[3, 5, 6, 7, 77, 100, 499]]).all() and int(torch.isnan(out).sum()) == 7 * 8
    assert torch.isfinite(torch.autograd.grad(out, w, torch.ones_like(out))[0]).all()
    assert torch.equal(ops.embedding(torch.tensor([1.9, -0.5], device=DEV), w), w[[1, 0]])   # cut towards zero


@pytest.mark.parametrize("rows", [16, 700])
def test_embedding_padding_row(ops, rows):
    t = tokens_of(4000, rows)
    t[::3] = 5
    check_embedding(ops, t, table(rows, 8), padding_idx=5)
    check_embedding(ops, t, table(rows, 8), padding_idx=5 - rows)
    check_embedding(ops, torch.full((64,), 5, device=DEV), table(rows, 8), padding_idx=5)


@pytest.mark.parametrize("rows", [16, 700])
def test_embedding_values_that_are_not_finite_stay_in_their_rows(ops, rows):
    t = tokens_of(3000, rows)
    w = table(rows, 8)
    w[3, 2], w[4, 1] = math.inf, math.nan
    out = ops.embedding(t, w.requires_grad_())
    g = torch.ones_like(out)
    at = int((t == 9).nonzero()[0])
    g[at, 0], g[at, 1] = math.inf, math.nan
    dw, = torch.autograd.grad(out, w, g)
    assert not torch.isfinite(dw[9, :2]).any() and int((~torch.isfinite(dw)).sum()) == 2


def test_embedding_views_and_addresses(ops):
    """weights and gradients that begin anywhere, transposed and strided views, tokens of a slice"""
    buf = torch.randn(16 * 6 + 3, generator=gen(1)).to(DEV)
    t = tokens_of(999, 16)
    for at in range(4):
        check_embedding(ops, t, buf[at:at + 96].view(16, 6))
        check_embedding(ops, t, buf.to(BF16)[at:at + 96].view(16, 6))
    check_embedding(ops, t[::3], table(6, 16).t())
    check_embedding(ops, t.view(27, 37).t(), table(64, 8)[::4, 2:])
    w = table(1000, 10).requires_grad_()
    t = tokens_of(3000, 1000)
    g = torch.randn(10, 3000, generator=gen(5)).to(DEV)
    got, = torch.autograd.grad(ops.embedding(t, w), w, g.t())
    want, = torch.autograd.grad(ops.embedding(t, w), w, g.t().contiguous())
    assert torch.equal(got, want)
    ops.embedding(t, w).sum().backward()   # the gradient is one expanded value
    assert torch.equal(w.grad, torch.bincount(t, minlength=1000).float()[:, None].expand(1000, 10))


def test_embedding_offsets_past_32_bits(ops):
    """2^31 values and more in the output and in the table"""
    w = torch.zeros(2 ** 21 + 2, 1024, dtype=BF16, device=DEV)
    w[-1] = 3.0
    t = torch.full((2 ** 21 + 5,), 2 ** 21 + 1, dtype=torch.int64, device=DEV)
    t[0] = 0
    w.requires_grad_()
    out = ops.embedding(t, w, scale=2.0)
    assert float(out[-1, -1].detach()) == 6.0 and float(out[1, 0].detach()) == 6.0 and float(out[0, 5].detach()) == 0.0
    assert bool((out[1:] == 6.0).all())
    g = torch.zeros_like(out)
    g[-1, -1] = 1.0
    dw, = torch.autograd.grad(out, w, g)
    assert float(dw[-1, -1]) == 2.0 and int((dw != 0).sum()) == 1


def test_embedding_scales(ops):
    """any finite float32, a tensor of one value among them; one that is finite in 64 bits alone would make every row infinite"""
    t, w = tokens_of(50, 16), table(16, 4)
    for scale in (0.0, -2.5, 1e-30, 1e30, torch.tensor(0.75)):
        check_embedding(ops, t, w, scale=float(scale))
        assert torch.equal(ops.embedding(t, w, scale=scale), ops.embedding(t, w, scale=float(scale)))
    assert torch.isfinite(ops.embedding(t, w * 0.01, scale=3.4028234e38)).all()
    for scale in (1e39, -1e300, math.inf, math.nan):
        with pytest.raises(ValueError, match="finite in float32"):
            ops.embedding(t, w, scale=scale)


def test_embedding_of_tokens_along_two_axes_of_a_grid(ops):
    """more workgroups than one axis takes, forward and where the runs are joined; sums of small whole numbers are exact"""
    n = 2 ** 25 + 7
    t, w = torch.randint(0, 1000, (n,), device=DEV, dtype=torch.int32), torch.randn(1000, 33, device=DEV).to(BF16)
    out = ops.embedding(t, w)
    for part in (slice(0, 4000), slice(n - 4000, n)):
        assert torch.equal(out[part], w[t[part].long()])
    del out
    n = 2 ** 27 + 77
    t = torch.randint(0, 20000, (n,), device=DEV, dtype=torch.int32)
    t[-3000:] = 19999
    w = torch.zeros(20000, 1, device=DEV, requires_grad=True)
    g = torch.randint(-1, 2, (n, 1), device=DEV).float()
    dw, = torch.autograd.grad(ops.embedding(t, w), w, g)
    want = torch.bincount(t[g[:, 0] == 1], minlength=20000) - torch.bincount(t[g[:, 0] == -1], minlength=20000)
    assert torch.equal(dw[:, 0].long(), want)


# ---- cross entropy ----------------------------------------------------------------------------------------------------------------
def check_loss(ops, logits, labels, weight=None, ignore_index=-100, reduction="mean", upstream=None):
    """logits on the GPU.  Per row: e^(x - m) is off by 2^-22 and |x - m| 2^-23 of itself, a sum of them by at most 64 additions in
    a row (64 U); for the differences here (below 60, or so small that nothing is left of them) 2^-16 covers both.  So the sum's logarithm is off
    by 2^-16, m - x by U |m - x|, and a probability p by 2^-16 p."""
    x = logits.detach().requires_grad_()
    loss = ops.cross_entropy(x, labels, weight=weight, ignore_index=ignore_index, reduction=reduction)
    assert loss.dtype == F32
    xd, y = logits.detach().double().cpu(), labels.cpu().long()
    n, c = xd.shape
    live, inside = y != ignore_index, (y >= 0) & (y < c)
    at = torch.where(inside, y, 0)
    w = (torch.ones(n, dtype=torch.float64) if weight is None else weight.double().cpu()[at])
    w = torch.where(live, torch.where(inside, w, math.nan), 0.0)
    lp = torch.log_softmax(xd, 1)
    lp[torch.isinf(xd).all(1)] = math.nan
    own = -lp.gather(1, at[:, None])[:, 0]
    rows = torch.where(live, w * own, 0.0)
    total = w.sum()
    m = xd.max(1).values
    slack = 2.0 ** -16 + U * (m - xd.gather(1, at[:, None])[:, 0]).abs()
    slack = torch.where(live & torch.isfinite(slack), w.abs() * (slack + 2 * U * own.abs()), 0.0)
    if reduction == "none":
        close(loss, rows, slack + rounding(rows, F32), "loss")
        k = w * (1.0 if upstream is None else upstream.double().cpu())
    else:
        want = rows.sum() / (total if reduction == "mean" else 1.0)
        close(loss, want, slack.sum() / (total if reduction == "mean" else 1.0) + rounding(want, F32), "loss")
        k = w / (total if reduction == "mean" else 1.0) * (1.0 if upstream is None else float(upstream))
    g = torch.ones_like(loss) if upstream is None else upstream.to(loss.device)
    dx, = torch.autograd.grad(loss, x, g, retain_graph=True)
    assert dx.dtype == logits.dtype
    p = lp.exp()
    hot = torch.zeros_like(p)
    hot[torch.arange(n), at] = inside.double()
    want = torch.where(live[:, None], k[:, None] * (p - hot), 0.0)
    bound = torch.where(live[:, None], k.abs()[:, None] * (p * 2.0 ** -16 + 4 * U), 0.0)
    close(dx, want, bound + rounding(want, logits.dtype), "gradient")
    again, = torch.autograd.grad(loss, x, g)   # of the retained graph: computed from the logits
    assert torch.equal(again.nan_to_num(7.0), dx.nan_to_num(7.0))
    with torch.no_grad():
        assert torch.equal(ops.cross_entropy(x, labels, weight=weight, ignore_index=ignore_index, reduction=reduction).nan_to_num(7.0),
                           loss.detach().nan_to_num(7.0))


def logits_of(n, c, dtype=F32, seed=1, scale=3.0):
    return (torch.randn(n, c, generator=gen(seed)) * scale).to(dtype).to(DEV)


def labels_of(n, c, dtype=torch.int64, seed=2):
    return torch.randint(0, c, (n,), generator=gen(seed)).to(dtype).to(DEV)


CLASSES = [1, 2, 3, 4, 5, 16, 17, 64, 65, 255, 256, 257, 1000, 2047, 2048, 4100, 8193, 16385, 33000]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("c", CLASSES)
def test_loss_classes(ops, c, dtype):
    n = 37 if c < 5000 else 5
    check_loss(ops, logits_of(n, c, dtype), labels_of(n, c))
    check_loss(ops, logits_of(n, c, dtype), labels_of(n, c), weight=torch.rand(c, generator=gen(4)).to(DEV) + 0.1, reduction="sum")


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 257, 512, 5000, 70001])
def test_loss_rows(ops, n):
    check_loss(ops, logits_of(n, 2), labels_of(n, 2), weight=torch.tensor([1.0, 1.7], device=DEV))
    if n < 6000:
        check_loss(ops, logits_of(n, 300, BF16), labels_of(n, 300, torch.int32))


@pytest.mark.parametrize("c", [2, 70, 300, 40001])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_reductions_labels_and_upstream(ops, c, reduction):
    n = 33
    x, y = logits_of(n, c), labels_of(n, c)
    y[::4] = -100
    up = torch.rand(n, generator=gen(8)) + 0.5 if reduction == "none" else torch.tensor(0.37)
    check_loss(ops, x, y, reduction=reduction)
    check_loss(ops, x, y, reduction=reduction, upstream=up)
    check_loss(ops, x, y % c, ignore_index=1, reduction=reduction, weight=torch.rand(c, generator=gen(3)).to(DEV), upstream=up)
    if c <= 256:
        check_loss(ops, x, (y % c).to(torch.uint8), ignore_index=0, reduction=reduction)


@pytest.mark.parametrize("c", [2, 100, 300, 9001, 40001])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_loss_values_at_the_edges(ops, c, dtype):
    """masked classes (-inf, the lowest value), rows with nothing left, NaN and inf in rows that count and in rows that do not"""
    n = 12
    x, y = logits_of(n, c, dtype), torch.zeros(n, dtype=torch.int64, device=DEV)
    low = torch.finfo(dtype).min
    x[0, 1:] = -math.inf                  # one class is left
    x[1, :] = -math.inf                   # none is
    x[2, 1:] = low
    x[3, :] = low                         # all equal
    x[4, c - 1] = math.nan
    x[5, c - 1] = math.inf
    x[6, :] = math.nan
    x[7, :] = -math.inf
    x[8, 0] = -math.inf                   # its own class is impossible: an infinite loss
    y[6], y[7] = -100, -100
    x[9, :] = torch.finfo(dtype).max / 4
    if c > 2:
        x[10, : c // 2 + 1] = -math.inf   # whole accesses of a thread
        y[10] = c - 1
    xd = x.double().cpu()
    loss = ops.cross_entropy(x.requires_grad_(), y, reduction="none")
    want = torch.nn.functional.cross_entropy(xd, y.cpu(), reduction="none")
    assert torch.equal(torch.isnan(loss.cpu()), torch.isnan(want)) and torch.isnan(want[[1, 4, 5]]).all()
    fine = torch.isfinite(want)
    assert math.isinf(float(loss[8].detach())) and float(loss[6].detach()) == 0.0 == float(loss[7].detach())
    assert (loss.detach().double().cpu()[fine] - want[fine]).abs().max() < 2.0 ** -15
    dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    dx = dx.double().cpu()
    assert (dx[[6, 7]] == 0).all()
    for r in (0, 2, 3, 8, 9, 10):
        p = torch.softmax(xd[r], 0)
        p[y[r]] -= 1
        assert (dx[r] - p).abs().max() < 2.0 ** -15 + torch.finfo(dtype).eps
    assert torch.isnan(dx[[1, 4, 5]]).any(1).all()
    # the same rows by the mean of the sound ones: what is ignored does not count
    y2 = y.clone()
    y2[[1, 4, 5, 8]] = -100
    mean = ops.cross_entropy(x, y2)
    assert abs(float(mean.detach()) - float(want[[0, 2, 3, 9, 10, 11]].mean())) < 2.0 ** -15
    assert torch.isfinite(torch.autograd.grad(mean, x)[0]).all()


def test_loss_nothing_to_count(ops):
    x = logits_of(4, 5).requires_grad_()
    y = torch.full((4,), -100, device=DEV)
    loss = ops.cross_entropy(x, y)
    assert math.isnan(float(loss.detach())) and (torch.autograd.grad(loss, x)[0] == 0).all()
    assert float(ops.cross_entropy(x, y, reduction="sum").detach()) == 0.0
    e = torch.zeros(0, 5, device=DEV, requires_grad=True)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    assert math.isnan(float(ops.cross_entropy(e, none).detach())) and float(ops.cross_entropy(e, none, reduction="sum").detach()) == 0.0
    assert ops.cross_entropy(e, none, reduction="none").shape == (0,)
    assert torch.autograd.grad(ops.cross_entropy(e, none, reduction="sum"), e)[0].shape == (0, 5)


@pytest.mark.parametrize("c", [6, 500])
def test_loss_labels_outside_the_classes(ops, c):
    x, y = logits_of(6, c), labels_of(6, c)
    y[1], y[4] = c, -1
    check_loss(ops, x, y, reduction="none")
    loss = ops.cross_entropy(x.requires_grad_(), y)
    assert math.isnan(float(loss.detach()))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_loss_views_and_addresses(ops, dtype):
    """rows that begin anywhere, row strides, a transposed view, an expanded row; the gradient's rows at other places than the logits'"""
    big = logits_of(40, 700, dtype)
    y = labels_of(40, 600)
    for at in range(3):
        check_loss(ops, big[:, at:at + 601], y)
    check_loss(ops, big[::2, 5:], y[::2])
    check_loss(ops, big.t(), labels_of(700, 40))
    check_loss(ops, big[:1].expand(40, 700), y)
    flat = logits_of(1, 9 * 301 + 7, dtype)[0]
    for at in range(1, 8, 2):
        check_loss(ops, flat[at:at + 9 * 301].view(9, 301), labels_of(9, 301))


def test_loss_large_values_keep_their_probabilities(ops):
    """logits of 1e4 and more: a probability computed through a rounded log sum exp would be off by |lse| U = 6e-4 of itself"""
    for c in (2, 300, 40001):
        x = (torch.rand(8, c, generator=gen(4)) * 4 + 30000).to(DEV).requires_grad_()
        y = labels_of(8, c)
        dx, = torch.autograd.grad(ops.cross_entropy(x, y, reduction="sum"), x)
        p = torch.softmax(x.detach().double().cpu(), 1)
        p[torch.arange(8), y.cpu()] -= 1
        assert ((dx.double().cpu() - p).abs() / (p.abs() + 1e-9)).max() < 2.0 ** -15


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c", [20, 32, 33, 63, 64, 129, 200, 256, 1020, 1021, 2040, 2041, 2044, 2045, 4088, 4089, 4096, 4097])
def test_loss_rows_by_groups_of_lanes(ops, c, dtype):
    """rows for which one workgroup is too few, classes around each number of lanes and accesses; rows beginning anywhere"""
    n = 1100 if c < 300 else 9
    x, y = logits_of(n, c + 3, dtype), labels_of(n, c)
    y[::7] = -100
    check_loss(ops, x[:, 3:], y)
    check_loss(ops, x[:, :c].contiguous(), y, reduction="none", upstream=torch.randn(n, generator=gen(5)))


@pytest.mark.parametrize("n, c", [(600001, 20), (2200001, 40), (70001, 700), (17001, 5000)])
def test_loss_of_many_rows_is_the_sum_of_its_rows(ops, n, c):
    """more sums than one workgroup joins: they are the rows' losses added in 64 bits, rounded once (and the mean's quotient with them)"""
    x = torch.randn(n, c, device=DEV, dtype=BF16)
    y = torch.randint(0, c, (n,), device=DEV)
    rows = ops.cross_entropy(x, y, reduction="none").double()
    total = float(rows.cpu().sum())
    assert abs(float(ops.cross_entropy(x, y, reduction="sum")) - total) <= total * U * 1.001
    assert abs(float(ops.cross_entropy(x, y)) - total / n) <= total / n * U * 1.001
    loss = ops.cross_entropy(x.requires_grad_(), y)
    assert abs(float(loss.detach()) - total / n) <= total / n * U * 1.001


@pytest.mark.parametrize("n, c, more", [(2 ** 21 + 3, 4099, 1), (2 ** 23 + 5, 1021, 1), (2 ** 26 + 9, 30, 0)])
def test_loss_of_rows_along_two_axes_of_a_grid(ops, n, c, more):
    """more workgroups than one axis takes: the rows at the end are what they are by themselves"""
    x = torch.randn(1, c + more, device=DEV).to(BF16).expand(n, c + more).contiguous()
    x[-4000:] = torch.randn(4000, c + more, device=DEV).to(BF16)
    x = x[:, :c]
    y = torch.randint(0, c, (n,), device=DEV)
    x.requires_grad_()
    loss = ops.cross_entropy(x, y, reduction="none")
    dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    for part in (slice(0, 4000), slice(n - 4000, n)):
        e = x.detach()[part].requires_grad_()
        l = ops.cross_entropy(e, y[part], reduction="none")
        assert torch.equal(l, loss[part]) and torch.equal(torch.autograd.grad(l, e, torch.ones_like(l))[0], dx[part])


@pytest.mark.parametrize("n, c, dtype", [(40, 2, F32), (300, 300, BF16), (7, 40001, F32)])
@pytest.mark.parametrize("forward", ["eager", "captured apart"])
def test_loss_backward_captured_by_itself(ops, n, c, dtype, forward):
    """replayed under one upstream gradient after another: each replay is the gradient for its own, whatever the one before it was"""
    x, y = logits_of(n, c, dtype), labels_of(n, c)
    ups = [1.0, 2.0, 1.0, 0.25, 1.0]
    want = []
    for u in ups:
        leaf = x.clone().requires_grad_()
        want.append(torch.autograd.grad(ops.cross_entropy(leaf, y), leaf, torch.tensor(u, device=DEV))[0])
    leaf, up = x.clone().requires_grad_(), torch.ones((), device=DEV)
    side, first, second = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.cross_entropy(leaf, y), leaf, up)
        if forward == "eager":
            loss = ops.cross_entropy(leaf, y)
    torch.cuda.synchronize()
    if forward != "eager":
        with torch.cuda.graph(first, stream=side):
            loss = ops.cross_entropy(leaf, y)
    with torch.cuda.graph(second, stream=side):
        dx, = torch.autograd.grad(loss, leaf, up)
    if forward != "eager":
        first.replay()
    for u, w in zip(ups, want):
        up.fill_(u)
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, w), u


# ---- the norm of gradients ---------------------------------------------------------------------------------------------------------
def check_clip(ops, grads, max_norm, out_dtype=None):
    """the norm is rounded once; an output is the gradient times a factor in 64 bits, rounded to 32 bits and to its type"""
    gd = [g.double().cpu() for g in grads]
    norm = math.sqrt(sum(float((g * g).sum()) for g in gd))
    k = min(1.0, max_norm / (norm + 1e-6))
    out = None if out_dtype is None else [torch.full(g.shape, 9.0, dtype=out_dtype, device=DEV) for g in grads]
    keep = [g.clone() for g in grads]
    got, outs = ops.clip_grad_norm(grads, max_norm, out=out)
    assert abs(float(got) - norm) <= norm * 2 * U and got.dtype == F32 and got.shape == ()
    assert float(ops.grad_norm(grads)) == float(got)
    for g, o, a, b in zip(gd, outs, grads, keep):
        close(o, g * k, rounding(g * k, o.dtype) + 2 * U * (g * k).abs())
        assert torch.equal(a, b)
    # in place
    params = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g.clone() if g.is_contiguous() else g
    assert float(ops.clip_grad_norm_(params, max_norm)) == float(got)
    for p, g in zip(params, gd):
        close(p.grad, g * k, rounding(g * k, p.grad.dtype) + 2 * U * (g * k).abs())


@pytest.mark.parametrize("cut", [0.1, 0.999, 1.5])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_clip_sizes(ops, dtype, cut):
    sizes = [1, 2, 3, 7, 8, 9, 4095, 4096, 4097, 16384 * 3 + 5, 100003]
    grads = [torch.randn(n, generator=gen(n)).to(dtype).to(DEV) for n in sizes]
    norm = math.sqrt(sum(sizes))
    check_clip(ops, grads, cut * norm)
    check_clip(ops, grads, cut * norm, out_dtype=F32)
    for g in grads:
        check_clip(ops, [g], cut * math.sqrt(g.numel()))


@pytest.mark.parametrize("count", [1, 2, 95, 96, 97, 193, 500])
def test_clip_many_tensors_of_every_type(ops, count):
    grads = [torch.randn(3 + 17 * i % 91, 1 + i % 5, generator=gen(i)).to((F32, BF16, F16)[i % 3]).to(DEV) for i in range(count)]
    check_clip(ops, grads, 0.25 * math.sqrt(sum(g.numel() for g in grads)))
    check_clip(ops, grads, 0.25, out_dtype=F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_clip_tensors_that_begin_anywhere(ops, dtype):
    """views of one buffer, as a bucket of gradients has them, and outputs at other places within 16 bytes"""
    flat = torch.randn(60000, generator=gen(1)).to(dtype).to(DEV)
    sizes = [1, 2, 3, 5, 20000, 13, 8, 30001, 64]
    grads = list(flat[:sum(sizes)].split(sizes))
    for out_dtype in (dtype, F32):
        for at in range(4):
            place = torch.full((sum(sizes) + 9,), 9.0, dtype=out_dtype, device=DEV)
            norm, outs = ops.clip_grad_norm(grads, 20.0, out=list(place[at:at + sum(sizes)].split(sizes)))
            want = flat[:sum(sizes)].double().cpu()
            want = want * (20.0 / (float(want.norm()) + 1e-6))
            close(place[at:at + sum(sizes)], want, rounding(want, out_dtype) + 2 * U * want.abs())
            assert (place[:at] == 9).all() and (place[at + sum(sizes):] == 9).all()   # nothing beside them


def test_clip_orders_and_strides(ops):
    g = torch.randn(40, 30, generator=gen(1)).to(DEV)
    check_clip(ops, [g.t(), g[:, ::2], g[:0], torch.randn(2, 3, 4, 5, generator=gen(2)).to(DEV).permute(3, 0, 2, 1)], 3.0)
    p = torch.nn.Parameter(torch.zeros(30, 40, device=DEV))
    p.grad = g.t()
    ops.clip_grad_norm_(p, 1.0)           # a tensor itself, as torch takes it
    close(g, (w := torch.randn(40, 30, generator=gen(1)).double()) / (w.norm() + 1e-6), 2.0 ** -22)


def test_clip_outputs_over_strided_gradients(ops):
    """a transposed gradient and one with gaps are copied for the kernels; an output over the gradient itself is refused all the same,
    and none of its values has changed"""
    buf = torch.randn(40, 30, generator=gen(1)).to(DEV)
    keep = buf.clone()
    for g, o in ((buf.t(), buf.view(30, 40)), (buf[:, ::2], buf.view(-1)[:600].view(40, 15)), (buf[1:, :10], buf.view(-1)[700:1090].view(39, 10))):
        with pytest.raises(ValueError, match="overlaps a gradient"):
            ops.clip_grad_norm([g], 1.0, out=[o])
        assert torch.equal(buf, keep)
    norm, (o,) = ops.clip_grad_norm([buf[:20, ::2]], 1.0, out=[buf.view(-1)[600:900].view(20, 15)])   # behind it
    want = keep[:20, ::2].double().cpu()
    close(o, want / (want.norm() + 1e-6), 2.0 ** -22)
    assert torch.equal(buf[:20], keep[:20])


def test_clip_values_at_the_edges(ops):
    big = [torch.full((100,), 3e38, device=DEV), torch.full((7,), -1e30, device=DEV)]
    norm, out = ops.clip_grad_norm(big, 1.0)
    assert math.isinf(float(norm)) or abs(float(norm) / 3e39 - 1) < 1e-6   # 3e39 is no float32
    assert float(ops.grad_norm([torch.full((9,), 1e30, device=DEV)])) == pytest.approx(3e30, rel=1e-6)   # its squares are none
    assert float(ops.grad_norm([torch.full((16,), 1e-30, device=DEV)])) == pytest.approx(4e-30, rel=1e-6)
    close(out[0], torch.full((100,), 0.1, dtype=torch.float64), 1e-6)
    for bad in (math.nan, math.inf):
        g = torch.ones(5000, device=DEV)
        g[4321] = bad
        p = torch.nn.Parameter(torch.zeros(5000, device=DEV))
        p.grad = g.clone()
        with pytest.raises(RuntimeError, match="not finite"):
            ops.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
        assert torch.equal(p.grad.nan_to_num(5.0), g.nan_to_num(5.0))   # nothing was changed
        q = torch.nn.Parameter(torch.zeros(5000, device=DEV))
        q.grad = g.clone()
        a, b = ops.clip_grad_norm_([p], 1.0), torch.nn.utils.clip_grad_norm_([q], 1.0)
        assert torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) and torch.equal(p.grad.nan_to_num(5.0), q.grad.nan_to_num(5.0))
    z = torch.zeros(10, device=DEV)
    norm, out = ops.clip_grad_norm([z], 0.0)
    assert float(norm) == 0.0 and (out[0] == 0).all()


def test_clip_nothing_shared_and_missing_gradients(ops):
    p, q, r = (torch.nn.Parameter(torch.zeros(50, device=DEV)) for _ in range(3))
    assert float(ops.clip_grad_norm_([p, q], 1.0)) == 0.0
    p.grad = torch.full((50,), 2.0, device=DEV)
    r.grad = p.grad                       # shared: counted and scaled once
    n = ops.clip_grad_norm_([p, q, r], 1.0)
    assert float(n) == pytest.approx(math.sqrt(200), rel=1e-6)
    close(p.grad, torch.full((50,), 2 / (math.sqrt(200) + 1e-6), dtype=torch.float64), 1e-7)
    p.grad, r.grad = (b := torch.ones(90, device=DEV))[:50], b[40:]
    with pytest.raises(ValueError, match="overlap"):
        ops.clip_grad_norm_([p, r], 1.0)
    with pytest.raises(ValueError, match="overlaps a gradient"):
        ops.clip_grad_norm([b], 1.0, out=[b])
    with pytest.raises(ValueError, match="overlap in memory"):
        ops.clip_grad_norm([p.grad, p.grad], 1.0, out=[b[40:], b[40:]])
    p.grad = torch.ones(1, device=DEV).expand(50)
    with pytest.raises(ValueError, match="expanded"):
        ops.clip_grad_norm_([p], 1.0)


# ---- lstm ---------------------------------------------------------------------------------------------------------------------------
def lstm_case(B, T, I, H, dirs=2, seed=1, spread=1.0, states=True):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    k = spread / math.sqrt(H)
    ws = [((torch.rand(*s, generator=g) * 2 - 1) * k) for _ in range(dirs) for s in ((4 * H, I), (4 * H, H), (4 * H,), (4 * H,))]
    h0, c0 = (r(dirs, B, H), r(dirs, B, H)) if states else (None, None)
    return r(B, T, I), ws, h0, c0, (r(B, T, dirs * H), r(dirs, B, H), r(dirs, B, H))


def plain_lstm(x, ws, h0, c0):
    """torch.nn.LSTM's definition in the type of its inputs"""
    B, T, _ = x.shape
    H, dirs = ws[1].shape[1], len(ws) // 4
    ys, hn, cn = [], [], []
    for d in range(dirs):
        w_ih, w_hh, b_ih, b_hh = ws[4 * d:4 * d + 4]
        h = x.new_zeros(B, H) if h0 is None else h0[d]
        c = x.new_zeros(B, H) if c0 is None else c0[d]
        out = [None] * T
        for t in range(T)[::-1 if d else 1]:
            i, f, g, o = (x[:, t] @ w_ih.t() + b_ih + h @ w_hh.t() + b_hh).split(H, 1)
            c = f.sigmoid() * c + i.sigmoid() * g.tanh()
            h = o.sigmoid() * c.tanh()
            out[t] = h
        ys.append(torch.stack(out, 1))
        hn.append(h)
        cn.append(c)
    return torch.cat(ys, 2), torch.stack(hn), torch.stack(cn)


def near(got, want, tol, what):
    """by the 2-norm over all values"""
    got, want = got.detach().double().cpu(), want.detach()
    assert got.shape == want.shape, what
    off, size = float((got - want).norm()), float(want.norm())
    assert off <= tol * max(size, 1e-30) + (0 if size else 1e-30), "%s: off by %g of its norm, allowed %g" % (what, off / max(size, 1e-30), tol)


def check_lstm(ops, B, T, I, H, dirs=2, states=True, spread=1.0, seed=1, parts=(True, True, True)):
    """A product of length n in 32 bits is off by at most n U of the products' sizes, the gates by 8 U more; a step hands its errors to
    the next one, so the chain of T steps has T of them.  dW sums B T terms, whose errors are those of dz and otherwise independent: their
    root on top."""
    x, ws, h0, c0, grads = lstm_case(B, T, I, H, dirs, seed, spread, states)
    tol = (4 * H + I + 40) * (T + 1) * U + math.sqrt(B * T) * 4 * U
    dev = [None if t is None else t.to(DEV).requires_grad_() for t in (x, h0, c0)]
    wdev = [w.to(DEV).requires_grad_() for w in ws]
    wide = [None if t is None else t.double().requires_grad_() for t in (x, h0, c0)]
    wwide = [w.double().requires_grad_() for w in ws]
    got = ops.lstm(dev[0], wdev, dev[1], dev[2])
    want = plain_lstm(wide[0], wwide, wide[1], wide[2])
    for g, w, name in zip(got, want, ("y", "hn", "cn")):
        near(g, w, tol, name)
    with torch.no_grad():
        for g, a in zip(ops.lstm(dev[0], wdev, dev[1], dev[2]), got):
            assert torch.equal(g, a)
    use = [i for i in range(3) if parts[i]]
    gs = [grads[i] for i in use]
    ins = [t for t in dev if t is not None] + wdev
    names = [n for n, t in zip(("x", "h0", "c0"), dev) if t is not None] + ["%s %d" % (n, d) for d in range(dirs) for n in ("w_ih", "w_hh", "b_ih", "b_hh")]
    dgot = torch.autograd.grad([got[i] for i in use], ins, [g.to(DEV) for g in gs], retain_graph=True)
    dwant = torch.autograd.grad([want[i] for i in use], [t for t in wide if t is not None] + wwide, [g.double() for g in gs])
    for g, w, name in zip(dgot, dwant, names):
        near(g, w, 4 * tol, "gradient of " + name)
    again = torch.autograd.grad([got[i] for i in use], ins, [g.to(DEV) for g in gs])
    for a, b in zip(dgot, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("H", [1, 3, 4, 15, 16, 17, 32, 48, 100, 128])
@pytest.mark.parametrize("I", [1, 7, 16, 33])
def test_lstm_units_and_inputs(ops, H, I):
    check_lstm(ops, 5, 3, I, H)


@pytest.mark.parametrize("B", [1, 2, 15, 16, 17, 63, 64, 65, 200, 513])
@pytest.mark.parametrize("T", [1, 2, 13])
def test_lstm_batches_and_steps(ops, B, T):
    check_lstm(ops, B, T, 16, 24, seed=B)


@pytest.mark.parametrize("dirs", [1, 2])
@pytest.mark.parametrize("states", [True, False])
@pytest.mark.parametrize("parts", [(True, True, True), (True, False, False), (False, True, False), (False, False, True)])
def test_lstm_directions_states_and_gradients_given(ops, dirs, states, parts):
    check_lstm(ops, 9, 4, 11, 20, dirs=dirs, states=states, parts=parts)
    check_lstm(ops, 70, 1, 8, 16, dirs=dirs, states=states, parts=parts)


@pytest.mark.parametrize("B,T,I,H", [(512, 13, 7, 128), (512, 13, 16, 128), (300, 13, 256, 256), (130, 13, 512, 256), (2, 200, 20, 40), (1000, 5, 260, 132), (40, 6, 300, 520)])
def test_lstm_the_models_layers_and_long_sequences(ops, B, T, I, H):
    check_lstm(ops, B, T, I, H)


@pytest.mark.parametrize("B,T,I,H,dirs,states", [(1900, 2, 20, 528, 2, True), (1900, 3, 5, 528, 2, False), (3900, 2, 8, 528, 1, True), (4100, 3, 9, 112, 2, True),
                                                 (4100, 2, 16, 100, 2, True), (8200, 2, 4, 80, 1, False), (16500, 2, 4, 68, 2, True)])
def test_lstm_many_sequences(ops, B, T, I, H, dirs, states):
    """the forms of many sequences: tiles that end inside the batch and inside the units, with a last tile of 16 units"""
    check_lstm(ops, B, T, I, H, dirs=dirs, states=states)


@pytest.mark.parametrize("B,T,I,H,dirs", [(32, 13, 64, 128, 2), (9, 13, 7, 20, 2), (16, 1, 256, 256, 2), (130, 13, 512, 256, 2), (512, 13, 512, 256, 2), (512, 13, 16, 128, 1),
                                           (1100, 13, 30, 130, 1), (4096, 13, 64, 128, 2), (4096, 13, 48, 256, 2)])
def test_lstm_holds_32_bits(ops, B, T, I, H, dirs):
    """as check_lstm, with the errors' signs mixed, so that an operand rounded to 16 bits (2^-9 of itself and more) or a product in fewer than
    24 shows in every form.  A sum of n products of mixed sign is off by 0.41 n^1/2 U of itself (the partial sums' sizes grow with the root of
    their length, each addition is off by U 3^-1/2 of one), the gates' functions by 4 U.  h is a quarter of its gates' arguments in size: four
    times that.  A step hands on less than two thirds of its error: three times.  Twice all that for what is not average: 24 (0.41 n^1/2 + 4) U.
    A gradient goes through twice as many products, and through the forward's values twice: four times; dW's sum of B T of them on top."""
    x, ws, h0, c0, grads = lstm_case(B, T, I, H, dirs, seed=B + H)
    tol = 24 * (0.41 * math.sqrt(I + H + 2) + 4) * U
    leaves = [t.to(DEV).requires_grad_() for t in (x, h0, c0, *ws)]
    wide = [t.to(DEV).double().requires_grad_() for t in (x, h0, c0, *ws)]
    got, want = ops.lstm(leaves[0], leaves[3:], leaves[1], leaves[2]), plain_lstm(wide[0], wide[3:], wide[1], wide[2])
    for g, w, name in zip(got, want, ("y", "hn", "cn")):
        near(g, w.cpu(), tol, name)
    gs = [g.to(DEV) for g in grads]
    dgot, dwant = torch.autograd.grad(got, leaves, gs), torch.autograd.grad(want, wide, [g.double() for g in gs])
    for k, (g, w) in enumerate(zip(dgot, dwant)):
        near(g, w.cpu(), 4 * tol + (0.41 * math.sqrt(B * T) * U if k > 2 else 0), "gradient %d" % k)


@pytest.mark.parametrize("B,T,I,H,dirs", [(2044, 3, 16, 128, 2), (2045, 3, 16, 128, 2), (2100, 2, 7, 100, 2), (4090, 2, 5, 72, 1), (4093, 2, 16, 65, 1), (2046, 2, 4, 64, 2)])
def test_lstm_at_the_change_from_one_launch_to_steps(ops, B, T, I, H, dirs):
    check_lstm(ops, B, T, I, H, dirs=dirs)


def test_lstm_saturated_gates_and_large_inputs(ops):
    """weights six times as large; inputs of 1e6 (an un-normalised read), where every gate is 0 or 1"""
    check_lstm(ops, 33, 13, 16, 32, spread=6.0)
    x, ws, h0, c0, grads = lstm_case(20, 3, 16, 32)
    x = x * 1e6
    leaves = [t.to(DEV).requires_grad_() for t in (x, h0, c0, *ws)]
    outs = ops.lstm(leaves[0], leaves[3:], leaves[1], leaves[2])
    want = plain_lstm(x.double(), [w.double() for w in ws], h0.double(), c0.double())
    for g, w in zip(outs, want):
        assert torch.isfinite(g).all() and (g.detach().double().cpu() - w).abs().max() < 0.02   # a gate's input of 1e6 is off by up to 0.06: those near 0 are not settled
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(outs, leaves, [g.to(DEV) for g in grads]))


def test_lstm_a_sequence_in_pieces_is_the_sequence(ops):
    """the states of one call handed to the next: the same bits as one call for pieces of two steps and more.  A single step adds
    W_ih x to the other products in an order of its own: each order is off by at most check_lstm's bound, both by twice that"""
    x, ws, h0, c0, _ = lstm_case(18, 9, 12, 36, dirs=1)
    x, ws, h0, c0 = x.to(DEV), [w.to(DEV) for w in ws], h0.to(DEV), c0.to(DEV)

    def pieces(*cuts):
        got, h, c = [], h0, c0
        for a, b in zip((0,) + cuts, cuts + (9,)):
            o, h, c = ops.lstm(x[:, a:b], ws, h, c)
            got.append(o)
        return torch.cat(got, 1), h, c
    with torch.no_grad():
        whole = ops.lstm(x, ws, h0, c0)
        assert all(torch.equal(a, b) for a, b in zip(pieces(4, 6), whole))
        for cuts in ((4, 5, 6), tuple(range(1, 9))):
            for got, want in zip(pieces(*cuts), whole):
                near(got, want.double().cpu(), 2 * (4 * 36 + 12 + 40) * 10 * U, "pieces")


def test_lstm_not_finite_stays_in_its_sequence(ops):
    x, ws, h0, c0, grads = lstm_case(70, 4, 8, 16)
    x[5, 2, 3], x[66, 0, 0] = math.nan, math.inf
    leaves = [t.to(DEV).requires_grad_() for t in (x, h0, c0, *ws)]
    outs = ops.lstm(leaves[0], leaves[3:], leaves[1], leaves[2])
    clean = [i for i in range(70) if i not in (5, 66)]
    assert torch.isnan(outs[0][5]).any() and torch.isfinite(outs[0][clean]).all()
    dx = torch.autograd.grad(outs, leaves[0], [g.to(DEV) for g in grads])[0]
    assert torch.isfinite(dx[clean]).all()


def test_lstm_empty_batch_and_views(ops):
    x, ws, h0, c0, grads = lstm_case(6, 5, 10, 14)
    leaves = [w.to(DEV).requires_grad_() for w in ws]
    e = torch.zeros(0, 5, 10, device=DEV, requires_grad=True)
    y, hn, cn = ops.lstm(e, leaves)
    assert y.shape == (0, 5, 28) and hn.shape == (2, 0, 14) == cn.shape
    got = torch.autograd.grad(y.sum(), [e] + leaves)
    assert got[0].shape == e.shape and all((g == 0).all() for g in got[1:])
    want = ops.lstm(x.to(DEV), leaves, h0.to(DEV), c0.to(DEV))
    xt = x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)           # not contiguous
    off = [torch.empty(w.numel() + 1, device=DEV)[1:].view(w.shape).copy_(w) for w in ws]   # not aligned to 16 bytes
    for got in (ops.lstm(xt, leaves, h0.to(DEV), c0.to(DEV)), ops.lstm(x.to(DEV), off, h0.to(DEV), c0.to(DEV))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_lstm_of_rows_along_two_axes_of_a_grid(ops):
    """2^30 - 64 rows of inputs in both directions.  One unit: a gate's argument is four products and sums, off by 8 U of their size
    (below 2 here), the gates' functions by 4 U each, and a step hands what it is off by on, by no more than itself: 32 U a step"""
    B, T = 3933120, 273
    x = torch.randn(B, 1, 1, device=DEV).expand(B, T, 1) * torch.linspace(-1.0, 1.0, T, device=DEV)[:, None]
    _, ws, _, _, _ = lstm_case(1, 1, 1, 1, seed=4)
    with torch.no_grad():
        y, hn, cn = ops.lstm(x, [w.to(DEV) for w in ws])
    at = torch.cat([torch.arange(2000), torch.randint(0, B, (2000,), generator=gen(1)), torch.arange(B - 2000, B)])
    want = plain_lstm(x[at.to(DEV)].double().cpu(), [w.double() for w in ws], None, None)
    for got, w in zip((y[at.to(DEV)], hn[:, at.to(DEV)], cn[:, at.to(DEV)]), want):
        close(got, w, 32 * U * T)


# ---- linear ------------------------------------------------------------------------------------------------------------------------
def check_linear(ops, shape, inputs, outputs, bias=True, seed=1):
    """each value is a sum of n products: off by at most n U of the sum of their sizes, and once more by the bias"""
    g = gen(seed)
    x, w, b = torch.randn(*shape, inputs, generator=g), torch.randn(outputs, inputs, generator=g), torch.randn(outputs, generator=g) if bias else None
    gy = torch.randn(*shape, outputs, generator=g)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b) if t is not None]
    y = ops.linear(*leaves)
    xd, wd, gd = x.double().reshape(-1, inputs), w.double(), gy.double().reshape(-1, outputs)
    rows = xd.shape[0]
    close(y, (xd @ wd.t() + (b.double() if bias else 0)).view(*shape, outputs),
          (inputs + 1) * U * (xd.abs() @ wd.abs().t() + (b.double().abs() if bias else 0)).view(*shape, outputs) + 1e-30, "y")
    got = torch.autograd.grad(y, leaves, gy.to(DEV), retain_graph=True)
    close(got[0], (gd @ wd).view(*shape, inputs), outputs * U * (gd.abs() @ wd.abs()).view(*shape, inputs) + 1e-30, "dx")
    close(got[1], gd.t() @ xd, (rows + 1) * U * (gd.abs().t() @ xd.abs()) + 1e-30, "dw")
    if bias:
        close(got[2], gd.sum(0), (rows + 1) * U * gd.abs().sum(0) + 1e-30, "db")
    assert all(torch.equal(a, c) for a, c in zip(got, torch.autograd.grad(y, leaves, gy.to(DEV))))


@pytest.mark.parametrize("rows", [0, 1, 15, 64, 65, 130, 1000, 6656])
@pytest.mark.parametrize("inputs,outputs", [(1, 1), (7, 2), (16, 16), (256, 2), (33, 65), (512, 256), (256, 128)])
def test_linear_sizes(ops, rows, inputs, outputs):
    check_linear(ops, (rows,), inputs, outputs)



@pytest.mark.parametrize("rows, inputs, outputs", [(1, 4096, 700), (16, 1000, 1000), (17, 33, 16), (16385, 40, 16), (5000, 260, 1), (33, 300, 65),
                                                   (700, 31, 1500), (9000, 128, 130), (4, 12, 2000), (100, 2, 5000)])
def test_linear_few_rows_or_columns(ops, rows, inputs, outputs):
    """sums shared by waves, or in parts where the tiles are few; a part's end inside a tile"""
    check_linear(ops, (rows,), inputs, outputs)


def test_linear_shapes_views_and_missing_parts(ops):
    check_linear(ops, (3, 5, 7), 20, 12)
    check_linear(ops, (), 20, 12)
    check_linear(ops, (40,), 20, 12, bias=False)
    check_linear(ops, (70000,), 24, 36)
    check_linear(ops, (20000,), 300, 260)
    x, w, b = (torch.randn(*s, generator=gen(2)).to(DEV) for s in ((90, 48), (32, 48), (32,)))
    want = ops.linear(x, w, b)
    off = [torch.empty(t.numel() + 1, device=DEV)[1:].view(t.shape).copy_(t) for t in (x, w, b)]   # not aligned to 16 bytes
    assert torch.equal(ops.linear(*off), want)
    assert torch.equal(ops.linear(x.t().contiguous().t(), w.t().contiguous().t(), b), want)
    only = w.clone().requires_grad_()
    gw, = torch.autograd.grad(ops.linear(x, only, b).sum(), only)      # x needs no gradient; the gradient of y is one expanded value
    assert torch.allclose(gw, x.sum(0).expand(32, 48), rtol=2e-5, atol=2e-5)
    bad = x.clone()
    bad[7, 3] = math.nan
    y = ops.linear(bad, w, b)
    assert torch.isnan(y[7]).all() and int(torch.isnan(y).sum()) == 32


@pytest.mark.parametrize("inputs, outputs", [(2, 2), (4, 1)])
def test_linear_of_rows_along_two_axes_of_a_grid(ops, inputs, outputs):
    """2^29 rows and more; whole numbers, whose sums are exact"""
    rows = 2 ** 29 + 37
    whole = lambda *shape: torch.randint(-1, 2, shape, device=DEV, dtype=torch.int8).float()
    x, w, b = whole(rows, inputs), torch.tensor([[2.0, -3.0, 5.0, -7.0], [11.0, 13.0, -17.0, 19.0]], device=DEV)[:outputs, :inputs], torch.tensor([23.0, -29.0], device=DEV)[:outputs]
    x.requires_grad_()
    w, b = w.contiguous().requires_grad_(), b.clone().requires_grad_()
    y = ops.linear(x, w, b)
    with torch.no_grad():
        for o in range(outputs):
            want = torch.full((rows,), float(b[o]), device=DEV)
            for i in range(inputs):
                want += x[:, i] * float(w[o, i])
            assert torch.equal(y[:, o], want)
        del want
        g = whole(rows, outputs)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
        del y
        for i in range(inputs):
            assert torch.equal(dx[:, i], sum(g[:, o] * float(w[o, i]) for o in range(outputs)))
            for o in range(outputs):
                assert float(dw[o, i]) == float((g[:, o] * x[:, i]).sum(dtype=torch.float64))
        assert torch.equal(db.double(), g.sum(0, dtype=torch.float64))


@pytest.mark.parametrize("what", ["embedding", "loss", "lstm"])
def test_gradients_against_differences(ops, what):
    """f(v + e d) - f(v - e d) over 2 e along a random direction d: the difference quotient is off by e^2 of the third derivative, and by
    the function's own rounding over e -- with e = 2^-7 and values near 1 below 2^-10"""
    e, g = 2.0 ** -7, gen(6)
    if what == "embedding":
        t = tokens_of(60, 16)
        v = [table(16, 4)]
        f = lambda w: (ops.embedding(t, w, scale=1.5) * coef).sum()
        coef = torch.randn(60, 4, generator=g).to(DEV)
    elif what == "loss":
        y, wt = labels_of(12, 5), torch.rand(5, generator=g).to(DEV) + 0.5
        v = [logits_of(12, 5, scale=1.0)]
        f = lambda x: ops.cross_entropy(x, y, weight=wt)
    else:
        x, ws, h0, c0, gr = lstm_case(4, 3, 5, 6)
        v = [t.to(DEV) for t in (x, h0, c0, *ws)]
        gr = [t.to(DEV) / 10 for t in gr]
        f = lambda x, h, c, *w: sum((a * b).sum() for a, b in zip(ops.lstm(x, list(w), h, c), gr))
    v = [t.requires_grad_() for t in v]
    grads = torch.autograd.grad(f(*v), v)
    for k in range(len(v)):
        d = torch.randn(v[k].shape, generator=g).to(DEV)
        d /= d.norm()
        with torch.no_grad():
            hi, lo = (float(f(*[t + s * e * d if i == k else t for i, t in enumerate(v)])) for s in (1, -1))
        assert abs((hi - lo) / (2 * e) - float((grads[k] * d).sum())) < 2.0 ** -9
