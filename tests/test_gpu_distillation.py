"""GPU tests of the distillation loss and its gradient against the 64-bit oracle.

The bounds count roundings: a row's sum of exponentials is a chain of at most
vocab / 256 + 64 fp32 additions, an exponential of a difference x is off by
(|x| + 4) steps of fp32, a loss term by a few steps of its parts; the gradient is
rounded once to its type (half a step h)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import tree_oracle as orc

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda:0"
STEP = 2.0 ** -24


def np64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def inputs(rows, vocab, top, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * spread).to(dtype)
    y = torch.randn(rows, top, generator=g) * 2
    i = torch.randint(vocab, (rows, top), generator=g)
    return x, y, i


def check(mta, x, y, i, temperature=1.0, scale=1.0, name=""):
    """Forward and backward on the GPU against the oracle; returns the gradient."""
    leaf = x.to(DEV).requires_grad_(True)
    loss = mta.ops.topk_distillation(leaf, y.to(DEV), i.to(DEV), temperature=temperature)
    grad, = torch.autograd.grad(loss, leaf, torch.tensor(scale, device=DEV))
    assert loss.shape == () and loss.dtype == F32 and grad.shape == x.shape and grad.dtype == x.dtype
    vocab, top = x.shape[-1], y.shape[-1]
    x64, y64 = np64(x).reshape(-1, vocab), np64(y.float()).reshape(-1, top)
    ref, dref, e = orc.distillation(x64, y64, i.reshape(-1, top).numpy(), temperature)
    chain = (vocab / 256 + 64) * STEP
    far = np.where(np.isfinite(x64), x64.max(-1, keepdims=True) - x64, 0.0) / temperature
    yfar = float(np.where(np.isfinite(y64), y64.max() - y64, 0.0).max()) / temperature
    n = max(e["count"], 1)
    bound = temperature ** 2 / n * float((e["terms"] * (2 * chain + (16 + yfar) * STEP)).sum()) + STEP * abs(ref) + 1e-30
    assert abs(loss.item() - ref) <= bound, f"{name}: loss {loss.item()} against {ref}, bound {bound}"
    h = torch.finfo(x.dtype).eps / 2
    dref = dref * scale
    dbound = h * abs(dref) + scale * temperature / n * (
        e["q"] * (2 * chain + (2 * far + 16) * STEP) + e["p"] * ((top / 256 + 64 + 2 * yfar + 16) * STEP))
    dbound += {BF16: 2.0 ** -133, FP16: 2.0 ** -25, F32: 2.0 ** -126}[x.dtype]
    got = np64(grad).reshape(-1, vocab)
    worst = float((abs(got - dref) / dbound).max()) if got.size else 0.0
    assert worst <= 1.0, f"{name}: gradient error {worst:.2f} of its bound"
    return grad


@pytest.mark.parametrize("dtype,scale", [(BF16, 1.0), (FP16, 1024.0), (F32, -0.5)])
@pytest.mark.parametrize("rows,vocab,top,temperature", [
    (1, 1, 1, 1.0),
    (3, 7, 4, 2.0),
    (5, 8, 1, 1.0),
    (4, 300, 16, 0.5),
    (6, 1385, 64, 4.0),
    (3, 2047, 257, 1.0),
    (2, 2049, 1024, 1.5),
    (3, 16384, 64, 2.0),
    (2, 50001, 100, 1.0),
])
def test_distillation_matches_the_oracle(mta, dtype, scale, rows, vocab, top, temperature):
    x, y, i = inputs(rows, vocab, top, dtype, seed=rows + vocab)
    if rows > 2:
        i[1, top // 2:] = -1  # fewer entries
        i[2] = -100           # none
        y[0, :top // 2] = -math.inf
    check(mta, x, y, i, temperature, scale)


def test_rows_without_entries(mta):
    x, y, i = inputs(4, 33, 5, F32, 1)
    grad = check(mta, x, y, torch.full_like(i, -1))
    assert (grad == 0).all()
    leaf = x.to(DEV).requires_grad_(True)
    assert mta.ops.topk_distillation(leaf, torch.full_like(y, -math.inf).to(DEV), i.to(DEV)).item() == 0.0
    empty = torch.zeros(0, 33, device=DEV, requires_grad=True)
    loss = mta.ops.topk_distillation(empty, torch.zeros(0, 5, device=DEV), torch.zeros(0, 5, dtype=torch.int64, device=DEV))
    assert loss.item() == 0.0 and torch.autograd.grad(loss, empty)[0].shape == (0, 33)


def test_one_entry_is_cross_entropy(mta):
    """K = 1 puts all of the teacher's weight on one word."""
    x, y, i = inputs(50, 700, 1, F32, 2)
    leaf = x.to(DEV).requires_grad_(True)
    loss = mta.ops.topk_distillation(leaf, y.to(DEV), i.to(DEV))
    ref = torch.nn.functional.cross_entropy(x.double(), i[:, 0])
    assert abs(loss.item() - float(ref)) <= 1e-6 * float(ref)


def test_masked_words_and_large_logits(mta):
    """Words at -inf or the type's lowest value, and logits far from zero, where one logarithm would lose its bits."""
    x, y, i = inputs(6, 129, 4, F32, 3)
    i[:] = i % 40
    x[0, 40:] = -math.inf
    x[1, 40:] = torch.finfo(F32).min
    x[2] += 5000.0
    x[3] -= 5000.0
    check(mta, x, y, i)


def test_an_index_past_the_vocabulary_spoils_its_row_alone(mta):
    x, y, i = inputs(5, 40, 6, F32, 4)
    clean = check(mta, x, y, i)
    i[2, 3] = 40
    i[4, 1] = 1 << 40
    leaf = x.to(DEV).requires_grad_(True)
    loss = mta.ops.topk_distillation(leaf, y.to(DEV), i.to(DEV))
    grad, = torch.autograd.grad(loss, leaf)
    assert math.isnan(float(loss)) and grad[[2, 4]].isnan().all() and torch.equal(grad[[0, 1, 3]], clean[[0, 1, 3]])
    # a NaN among the teacher's logits, beside entries that are none
    i[2, 3], i[4, 1] = -1, -1
    y[1, 0] = math.nan
    i[1, 2] = -7
    loss = mta.ops.topk_distillation(leaf, y.to(DEV), i.to(DEV))
    grad, = torch.autograd.grad(loss, leaf)
    assert math.isnan(float(loss)) and grad[[0, 2, 3, 4]].isfinite().all() and grad[1].isnan().any()


@pytest.mark.parametrize("where", [slice(8, 16), slice(1000, 1001), slice(3, 4), slice(0, 1001)])
def test_a_logit_that_is_no_number_spoils_its_row_alone(mta, where):
    # alone in a thread, whole vectors of them, and beside -inf: the softmax over such a row is NaN everywhere
    x, y, i = inputs(4, 1001, 8, BF16, 15)
    x[1, where] = math.nan
    x[2, :] = -math.inf
    x[2, where] = math.nan
    i[1:3] = 500
    leaf = x.to(DEV).requires_grad_(True)
    loss = mta.ops.topk_distillation(leaf, y.to(DEV), i.to(DEV))
    grad, = torch.autograd.grad(loss, leaf)
    assert math.isnan(float(loss)) and grad[1:3].isnan().all() and grad[[0, 3]].isfinite().all()
    assert math.isnan(float(mta.ops.topk_distillation(x[1:2].to(DEV), y[1:2].to(DEV), i[1:2].to(DEV))))


@pytest.mark.parametrize("top", [64, 65, 300])
def test_entries_of_one_index_and_of_one_group(mta, top):
    """Every entry the same index; pairs and triples of it; and indexes 16384 apart or in one group of 8 columns."""
    vocab = 50001
    x, y, i = inputs(7, vocab, top, F32, 23)
    j = torch.arange(top)
    i[0] = 777
    i[1] = j // 2 * 100
    i[2] = j // 3 * 8 + 5
    i[3] = j % 3 * 16384 + j // 3 * 3
    i[4] = 40000 + j % 16
    i[5] = vocab - 1 - j % 2  # the columns past the last whole group
    i[6] = j
    check(mta, x, y, i, temperature=2.0)
    g = [torch.autograd.grad(mta.ops.topk_distillation(t, y.to(DEV), i.to(DEV)), t)[0]
         for t in (x.to(DEV).requires_grad_(True) for _ in range(3))]
    assert torch.equal(g[0], g[1]) and torch.equal(g[0], g[2])


def test_layouts_and_types_of_the_teacher(mta):
    x, y, i = inputs(12, 101, 8, BF16, 5)
    ref = check(mta, x, y.to(BF16), i, 2.0)
    # [2, 6, vocab] rows inside a wider buffer, off 16 bytes; a 16-bit teacher, int32 indices, other strides
    wide = torch.zeros(2, 6, 120, dtype=BF16, device=DEV)
    wide[..., 3:104] = x.to(DEV).view(2, 6, 101)
    leaf = wide[..., 3:104].detach().requires_grad_(True)
    t = torch.zeros(2, 6, 16, dtype=BF16, device=DEV)[..., ::2].copy_(y.view(2, 6, 8))
    loss = mta.ops.topk_distillation(leaf, t, i.view(2, 6, 8).to(DEV, torch.int32), temperature=2.0)
    grad, = torch.autograd.grad(loss, leaf)
    assert torch.equal(grad.view(12, 101), ref)
    turned = x.to(DEV).t().contiguous().t().requires_grad_(True)  # the vocabulary outermost
    loss = mta.ops.topk_distillation(turned, y.to(DEV, BF16), i.to(DEV), temperature=2.0)
    assert torch.equal(torch.autograd.grad(loss, turned)[0], ref)
    one = x[3].to(DEV).requires_grad_(True)  # a single row without leading dims
    loss = mta.ops.topk_distillation(one, y[3].to(DEV, BF16), i[3].to(DEV), temperature=2.0)
    assert torch.autograd.grad(loss, one)[0].shape == (101,)


def test_gradient_against_differences(mta):
    """Central differences of the operator's own loss along a direction u of unit size a word.  The remainder is at
    most h^2 / 6 times the third derivative (|u|^3 sums of probabilities: below 1 a row here), and the loss's own
    rounding 2 STEP |L| / h."""
    x, y, i = inputs(16, 50, 5, F32, 6)
    u = torch.randn(x.shape, generator=torch.Generator().manual_seed(7)).clamp(-1, 1).to(DEV)
    f = lambda t: mta.ops.topk_distillation(t, y.to(DEV), i.to(DEV), temperature=1.0).double()  # noqa: E731
    leaf = x.to(DEV).requires_grad_(True)
    grad, = torch.autograd.grad(f(leaf), leaf)
    h = 2.0 ** -6
    with torch.no_grad():
        diff = (f(leaf + h * u) - f(leaf - h * u)) / (2 * h)
        loss = float(f(leaf))
    assert abs(float(diff) - float((grad.double() * u.double()).sum())) <= h * h / 6 * 2 + 64 * STEP * (1 + abs(loss)) / h


def test_training_step_captured_and_repeated(mta):
    """Forward and backward recorded once and replayed on other inputs give the eager results, bit for bit; so does
    the same eager call twice."""
    x, y, i = (t.to(DEV) for t in inputs(64, 1385, 16, BF16, 8))

    def step(a, b, c):
        a = a.detach().requires_grad_(True)
        loss = mta.ops.topk_distillation(a, b, c, temperature=2.0)
        return loss.detach(), torch.autograd.grad(loss, a)[0]

    assert all(torch.equal(p, q) for p, q in zip(step(x, y, i), step(x, y, i)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, y, i)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x, y, i)
    for seed in (9, 10, 11):
        for t, s in zip((x, y, i), inputs(64, 1385, 16, BF16, seed)):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, step(x, y, i)))


def test_offsets_past_32_bits(mta):
    """More than 2^31 logits: the last rows are those of a call on them alone, scaled by the counts."""
    rows, vocab, top = 140_000, 16384, 3
    x = torch.zeros(rows, vocab, dtype=BF16, device=DEV)
    tail, y, i = (t.to(DEV) for t in inputs(4, vocab, top, BF16, 12))
    x[-4:] = tail
    index = torch.full((rows, top), -1, dtype=torch.int64, device=DEV)
    index[-4:] = i
    teacher = torch.zeros(rows, top, device=DEV)
    teacher[-4:] = y
    x.requires_grad_(True)
    loss = mta.ops.topk_distillation(x, teacher, index)
    grad, = torch.autograd.grad(loss, x)
    leaf = tail.detach().requires_grad_(True)
    ref = mta.ops.topk_distillation(leaf, y, i)
    assert torch.equal(loss, ref) and torch.equal(grad[-4:], torch.autograd.grad(ref, leaf)[0])
    assert not bool(grad[:-4].any())
