"""CPU tests of the oracle for drafted trees and distillation, and the refusals of their entry points."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import tree_oracle as orc
from tests import tree_refusals as refusals

BF16 = torch.bfloat16


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------
def test_ancestors_and_padding():
    assert orc.ancestors([-1, 0, 0, 2, -1, 4, 6, 5, 6, -2, 9, 3]) == [
        [0], [0, 1], [0, 2], [0, 2, 3], [4], [4, 5], None, [4, 5, 7], None, None, None, [0, 2, 3, 11]]


def test_a_chain_is_causal_attention():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, h, 11, 32, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    ref = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)[0, :, 6:].numpy()
    q, k, v = (x[0].numpy() for x in (q, k, v))
    out, mag, _ = orc.tree_attention(q[:, 6:], k[:, 6:], v[:, 6:], k[:, :6], v[:, :6], 6, [-1, 0, 1, 2, 3], 1 / math.sqrt(32))
    np.testing.assert_allclose(out, ref, rtol=1e-12, atol=1e-12)
    assert (mag >= abs(out) - 1e-12).all()


def test_rope_follows_the_depth():
    x = np.random.default_rng(0).normal(size=(2, 4, 8))
    freqs = np.outer(np.arange(9), 1.0 / 100.0 ** (np.arange(0, 8, 2) / 8))
    y, _ = orc.tree_rope(x, np.cos(freqs), np.sin(freqs), 5, [-1, 0, 0, -2])
    for n, pos in ((0, 5), (1, 6), (2, 6)):
        z = (x[:, n, 0::2] + 1j * x[:, n, 1::2]) * np.exp(1j * freqs[pos])
        np.testing.assert_allclose(y[:, n, 0::2] + 1j * y[:, n, 1::2], z, rtol=1e-12)
    assert (y[:, 3] == 0).all()


@pytest.mark.parametrize("drafted", [True, False])
def test_verification_keeps_the_targets_distribution(drafted):
    """The token after node 0, accepted or drawn, is a draw of the target's top-k softmax: 20000 walks, every
    frequency within 5 standard deviations.  A drafter's children are draws of its own softmax."""
    rng = np.random.default_rng(3)
    v, k, walks = 6, 4, 20000
    target, draft = rng.normal(size=(4, v)) * 1.5, rng.normal(size=(4, v)) * 1.5
    p, q = orc.top_softmax(target[0], k), orc.top_softmax(draft[0], k)
    parents, seen = [-1, 0, 0, 0], np.zeros(v)
    for _ in range(walks):
        tokens = [0, *(rng.choice(v, size=3, p=q) if drafted else (2, 5, 2))]
        path, token = orc.topk_verify(target, tokens, parents, rng.random(4), rng.exponential(size=v), k,
                                      draft if drafted else None)
        seen[tokens[path[1]] if len(path) > 1 else token] += 1
    assert (abs(seen - walks * p) <= 5 * np.sqrt(walks * p * (1 - p)) + 1e-9).all()


def test_distillation_against_autograd():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(5, 9, generator=g, dtype=torch.float64) * 2).requires_grad_(True)
    y = torch.randn(5, 4, generator=g, dtype=torch.float64)
    i = torch.tensor([[0, 3, 8, 3], [1, 2, -1, 4], [-1, -1, -1, -1], [5, 5, 5, 5], [7, 0, 6, -5]])
    t, rows = 1.7, [0, 1, 3, 4]
    loss = 0.0
    for r in rows:
        use = i[r] >= 0
        p = torch.softmax(y[r][use] / t, -1)
        loss = loss + (p * (p.log() - torch.log_softmax(x[r] / t, -1)[i[r][use]])).sum() * t * t / len(rows)
    loss.backward()
    got, grad, terms = orc.distillation(x.detach().numpy(), y.numpy(), i.numpy(), t)
    assert terms["count"] == 4 and abs(got - loss.item()) < 1e-12
    np.testing.assert_allclose(grad, x.grad.numpy(), rtol=1e-10, atol=1e-13)
    # the formula's gradient is that of the formula: central differences, third-order remainder 1e-10
    d = np.random.default_rng(0).normal(size=x.shape)
    f = lambda h: orc.distillation(x.detach().numpy() + h * d, y.numpy(), i.numpy(), t)[0]  # noqa: E731
    assert abs((f(1e-5) - f(-1e-5)) / 2e-5 - (grad * d).sum()) < 1e-8


# ---------------------------------------------------------------------------
# refusals: nothing is launched
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cases", [refusals.tree_attention, refusals.tree_rope_and_commit, refusals.topk_verify,
                                   refusals.topk_distillation], ids=lambda f: f.__name__)
def test_refusals(mta, cases):
    with FakeTensorMode():
        for err, match, call in cases(mta):
            with pytest.raises(err, match=match):
                call()


def _fake(*shape, dtype=BF16):
    return torch.empty(*shape, device="cuda", dtype=dtype)


def test_traced_calls_have_the_results_shapes(mta):
    with FakeTensorMode():
        q, k, v, kc, vc = refusals._nodes()
        par, length, cs = _fake(5, dtype=torch.int32), _fake(2, dtype=torch.int32), _fake(1, 1, 16, 32, dtype=torch.float32)
        assert mta.tree_attention(q, k, v, kc, vc, 7, par, repeats=2).shape == q.shape
        assert mta.tree_attention(q, k, v, kc, vc, length, par.expand(2, 5), repeats=2).shape == q.shape
        assert [t.shape for t in mta.tree_rope(q, k, cs, cs, 15, par)] == [q.shape, k.shape]
        path, count = _fake(2, 5, dtype=torch.int32), _fake(2, dtype=torch.int32)
        assert mta.tree_commit([k], [v], path, count, 3, [kc], [vc]) is None
        x, tok = _fake(2, 5, 40), _fake(2, 5, dtype=torch.int64)
        out = mta.ops.topk_verify(x, tok, par, _fake(2, 5, dtype=torch.float32), _fake(2, 40, dtype=torch.float32), 8,
                                  draft_logits=x)
        assert [(tuple(t.shape), t.dtype) for t in out] == [((2, 5), torch.int32), ((2,), torch.int32), ((2, 1), torch.int64)]
        y, i = _fake(2, 5, 7, dtype=torch.float32), _fake(2, 5, 7, dtype=torch.int64)
        assert mta.ops.topk_distillation(x, y, i, temperature=2.0).shape == ()


def test_cpu_tensors_are_refused(mta):
    x, n = torch.zeros(1, 2, 3, 64), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: mta.tree_attention(x, x, x, x, x, 1, n, repeats=1), lambda: mta.tree_rope(x, x, x, x, 1, n),
                 lambda: mta.tree_commit([x], [x], n, n, 1, [x], [x]),
                 lambda: mta.ops.topk_verify(x, n, n, n, n, 1), lambda: mta.ops.topk_distillation(x, x, n)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_c_entry_points_refuse(mta):
    """Every call fails (or has nothing to do) before a launch: the pointers are never followed."""
    lib = mta._native.load()
    p, i64 = 0x10000, ctypes.c_int64
    E_NULL, E_SHAPE, E_STRIDE, E_DTYPE, E_ROPE, E_WS = -1, -2, -3, -4, -5, -6

    def rope(q=p, s=(64, 64, 64, 1) * 2, rows=16, par=p, ps=0, ld=None, ls=0, length=3, b=1, hq=4, hkv=2, n=5, d=64, dt=0):
        return lib.mt_tree_rope(q, p, p, p, (i64 * 8)(*s), p, p, rows, par, ps, ld, ls, length, b, hq, hkv, n, d, dt, None)

    assert rope(q=None) == E_NULL and rope(par=None) == E_NULL
    assert rope(d=12) == E_SHAPE and rope(n=65) == E_SHAPE and rope(n=0) == E_SHAPE and rope(hq=5) == E_SHAPE
    assert rope(length=17) == E_SHAPE and rope(length=-1) == E_SHAPE and rope(rows=0) == E_ROPE
    assert rope(dt=3) == E_DTYPE and rope(ps=4) == E_STRIDE and rope(ld=p, ls=2) == E_STRIDE and rope(q=p + 2) == E_STRIDE
    assert rope(s=(64, 64, 65, 1) * 2) == E_STRIDE and rope(s=(64, 64, 64, 2) * 2) == E_STRIDE

    def attn(s=(64, 64, 64, 1) * 5, dt=0, d=64, n=5, length=7, cap=32, scale=0.1, ws=p, wsn=1 << 30, q=p, kc=p, o=p, hkv=2):
        return lib.mt_tree_attn(q, p, p, kc, p, o, (i64 * 20)(*s), p, 0, None, 0, length, cap, 2, 4, hkv, n, d, scale, dt, ws,
                                wsn, None)

    assert attn(dt=2) == E_DTYPE and attn(d=48) == E_SHAPE and attn(n=65) == E_SHAPE and attn(hkv=3) == E_SHAPE
    assert attn(length=33) == E_SHAPE and attn(cap=-1) == E_SHAPE and attn(scale=0.0) == E_SHAPE and attn(scale=math.nan) == E_SHAPE
    assert attn(q=None) == E_NULL and attn(kc=None) == E_NULL and attn(o=None) == E_NULL and attn(q=p + 8) == E_STRIDE
    assert attn(s=(64, 64, 64, 1) * 4 + (64, 64, 60, 1)) == E_STRIDE
    need = lib.mt_tree_attn_workspace_size(2, 4, 2, 5, 100_000, 64)
    assert need > 0 and need % 256 == 0 and lib.mt_tree_attn_workspace_size(2, 4, 3, 5, 100, 64) == 0
    assert attn(length=100_000, cap=100_000, wsn=need - 1) == E_WS and attn(length=100_000, cap=100_000, ws=None) == E_NULL

    one = (ctypes.c_void_p * 1)(p)

    def commit(layers=1, ptrs=one, s=(64, 64, 64, 1) * 4, dt=0, cap=32, path=p, n=5):
        return lib.mt_tree_commit(ptrs, one, one, one, layers, (i64 * 16)(*s), path, p, None, 0, 3, cap, 2, 2, n, 64, dt, None)

    assert commit(dt=2) == E_DTYPE and commit(path=None) == E_NULL and commit(ptrs=(ctypes.c_void_p * 1)(None)) == E_NULL
    assert commit(n=65) == E_SHAPE and commit(layers=-1) == E_SHAPE and commit(cap=2) == E_SHAPE
    assert commit(s=(64, 64, 64, 2) * 4) == E_STRIDE and commit(ptrs=(ctypes.c_void_p * 1)(p + 1)) == E_STRIDE
    assert commit(layers=0) == 0

    def verify(x=p, b=2, n=5, v=40, k=8, dt=0, ws=p, wsn=1 << 30, s=(200, 40, 200, 40), ps=0, ldn=40, tok=p):
        return lib.mt_topk_verify(x, None, (i64 * 4)(*s), tok, p, ps, p, p, ldn, p, p, p, b, n, v, k, dt, ws, wsn, None)

    assert verify(dt=3) == E_DTYPE and verify(n=65) == E_SHAPE and verify(v=32769) == E_SHAPE and verify(k=41) == E_SHAPE
    assert verify(x=None) == E_NULL and verify(tok=None) == E_NULL and verify(ws=None) == E_NULL and verify(x=p + 1) == E_STRIDE
    assert verify(ldn=39) == E_STRIDE and verify(ps=4) == E_STRIDE and verify(s=(200, -40, 0, 0)) == E_STRIDE
    assert verify(wsn=lib.mt_topk_verify_workspace_size(2, 5, 40, 8, 0) - 1) == E_WS
    assert verify(b=0) == 0

    def distill(x=p, ld=40, rows=3, v=40, k=7, t=1.0, state=p, dt=0):
        return lib.mt_topk_distill_fwd(x, ld, p, p, rows, v, k, t, state, p, dt, None)

    assert distill(dt=3) == E_DTYPE and distill(ld=39) == E_STRIDE and distill(rows=-1) == E_SHAPE and distill(v=0) == E_SHAPE
    assert distill(k=0) == E_SHAPE and distill(k=1025) == E_SHAPE and distill(t=0.0) == E_SHAPE and distill(t=math.inf) == E_SHAPE
    assert distill(x=None) == E_NULL and distill(x=p + 1) == E_STRIDE and distill(state=p + 4) == E_STRIDE
    assert lib.mt_topk_distill_bwd(p, 40, p, p, p, None, p, 3, 40, 7, 1.0, 0, None) == E_NULL
    assert lib.mt_topk_distill_bwd(None, 40, None, None, None, None, None, 0, 40, 7, 1.0, 0, None) == 0


# ---------------------------------------------------------------------------
# autograd rules, on meta tensors
# ---------------------------------------------------------------------------
def _meta(*shape, dtype=torch.float32, grad=False):
    return torch.empty(*shape, dtype=dtype, device="meta", requires_grad=grad)


def test_inference_operators_refuse_gradients(mta):
    mta._native.load()
    ops = torch.ops.mega_trading_amd
    par = _meta(5, dtype=torch.int32)
    q, k = (_meta(2, h, 5, 64, dtype=BF16, grad=True) for h in (4, 2))
    kc, cs = _meta(2, 2, 16, 64, dtype=BF16), _meta(16, 32)
    for out in (ops.tree_attn(q, k, k, kc, kc, None, 3, par, 0.1), ops.tree_rope(q, k, cs, cs, None, 3, par)[1]):
        assert out.requires_grad
        with pytest.raises(RuntimeError, match="no autograd formula"):
            torch.autograd.grad(out, (q, k), torch.ones_like(out), allow_unused=True)
    path, count = _meta(2, 5, dtype=torch.int32), _meta(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no autograd formula"):
        ops.tree_commit([k], [k], path, count, None, 3, [kc], [kc.clone()])
    kcs, vcs = [_meta(2, 2, 16, 64, dtype=BF16) for _ in range(2)], [_meta(2, 2, 16, 64, dtype=BF16) for _ in range(2)]
    before = [t._version for t in kcs + vcs]
    with torch.no_grad():
        ops.tree_commit([k, k], [k, k], path, count, None, 3, kcs, vcs)
    assert all(t._version > b for t, b in zip(kcs + vcs, before)), "the caches' versions count the write"


def test_distillation_gradient_rules(mta):
    mta._native.load()
    ops = torch.ops.mega_trading_amd
    x, y, i = _meta(3, 9, dtype=BF16, grad=True), _meta(3, 4, grad=True), _meta(3, 4, dtype=torch.int64)
    loss, state = ops.topk_distill_fwd(x, y, i, 2.0)
    assert loss.requires_grad and not state.requires_grad
    gx, gy = torch.autograd.grad(loss, (x, y), allow_unused=True, create_graph=True)
    assert gx.shape == x.shape and gx.dtype == BF16 and gy is None
    with pytest.raises(RuntimeError, match="no autograd formula"):
        torch.autograd.grad(gx, x, torch.ones_like(gx))
    with torch.no_grad():
        assert not ops.topk_distill_fwd(x, y, i, 2.0)[0].requires_grad
