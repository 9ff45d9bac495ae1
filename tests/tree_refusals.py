"""The calls that the drafted-tree operators and the distillation loss refuse, for traced tensors (CPU) and for
the GPU's (the checks are made in two places): (exception, message, call) for tensors made by torch.empty."""

from __future__ import annotations

import math

import torch

BF16 = torch.bfloat16


def _new(*shape, dtype=BF16):
    return torch.empty(*shape, device="cuda", dtype=dtype)


def _nodes(n=5, hq=4, hkv=2, d=64, b=2, cap=32, dtype=BF16):
    return [_new(b, h, m, d, dtype=dtype) for h, m in ((hq, n), (hkv, n), (hkv, n), (hkv, cap), (hkv, cap))]


def tree_attention(mta):
    par = _new(5, dtype=torch.int32)
    args = _nodes()
    return (
        (RuntimeError, "unsupported dtype", lambda: mta.tree_attention(*_nodes(dtype=torch.float32), 7, par, repeats=2)),
        (ValueError, "1 to 64 nodes", lambda: mta.tree_attention(*_nodes(n=65), 7, _new(65, dtype=torch.int32), repeats=2)),
        (ValueError, "1 to 64 nodes", lambda: mta.tree_attention(*_nodes(n=0), 7, _new(0, dtype=torch.int32), repeats=2)),
        (ValueError, "head_dim must be one of", lambda: mta.tree_attention(*_nodes(d=48), 7, par, repeats=2)),
        (ValueError, "multiplied by repeats", lambda: mta.tree_attention(*args, 7, par, repeats=4)),
        (ValueError, "query heads", lambda: mta.tree_attention(*_nodes(hq=3), 7, par, repeats=2)),
        (ValueError, "outside", lambda: mta.tree_attention(*args, 33, par, repeats=2)),
        (ValueError, "outside", lambda: mta.tree_attention(*args, -1, par, repeats=2)),
        (ValueError, "tensor length", lambda: mta.tree_attention(*args, _new(3, dtype=torch.int32), par, repeats=2)),
        (ValueError, "tensor length", lambda: mta.tree_attention(*args, _new(2, dtype=torch.int64), par, repeats=2)),
        (ValueError, "parents must be int32", lambda: mta.tree_attention(*args, 7, _new(5, dtype=torch.int64), repeats=2)),
        (ValueError, "parents must be int32", lambda: mta.tree_attention(*args, 7, _new(4, dtype=torch.int32), repeats=2)),
        (ValueError, "agree on batch", lambda: mta.tree_attention(args[0], *_nodes(n=6)[1:3], *args[3:], 7, par, repeats=2)),
        (ValueError, "caches must have the batch", lambda: mta.tree_attention(*args[:3], *_nodes(b=3)[3:], 7, par, repeats=2)),
        (ValueError, "too large", lambda: mta.tree_attention(*args[:3], *[t[:, :, :1].expand(2, 2, 1 << 33, 64) for t in args[3:]], 7, par, repeats=2)),
        (RuntimeError, "caches must have the dtype", lambda: mta.tree_attention(*args[:3], *_nodes(dtype=torch.float16)[3:], 7, par, repeats=2)),
    )


def tree_rope_and_commit(mta):
    q, k, v, kc, vc = _nodes()
    par, cs = _new(5, dtype=torch.int32), _new(1, 1, 16, 32, dtype=torch.float32)
    path, count = _new(2, 5, dtype=torch.int32), _new(2, dtype=torch.int32)
    return (
        (ValueError, "outside", lambda: mta.tree_rope(q, k, cs, cs, 16, par)),
        (ValueError, "head_dim/2", lambda: mta.tree_rope(q, k, cs[..., :31], cs, 3, par)),
        (ValueError, "multiple of 8", lambda: mta.tree_rope(_new(2, 4, 5, 20), _new(2, 2, 5, 20), cs, cs, 3, par)),
        (ValueError, "must have rows", lambda: mta.tree_rope(q, k, cs[:, :, :0], cs, 0, par)),
        (ValueError, "must have rows", lambda: mta.tree_rope(q, k, *[cs[:, :, :1].expand(1, 1, 1 << 32, 32)] * 2, 0, par)),
        (ValueError, "expanded", lambda: mta.tree_commit([k], [v], path, count, 3, [kc[:1].expand(2, -1, -1, -1)], [vc])),
        (ValueError, "one tensor per layer", lambda: mta.tree_commit([], [], path, count, 3, [], [])),
        (ValueError, "one tensor per layer", lambda: mta.tree_commit([k, k], [v], path, count, 3, [kc], [vc])),
        (ValueError, "share one shape", lambda: mta.tree_commit([k], [v[:, :, :4]], path, count, 3, [kc], [vc])),
        (ValueError, "path must be int32", lambda: mta.tree_commit([k], [v], path.long(), count, 3, [kc], [vc])),
        (ValueError, "count must be int32", lambda: mta.tree_commit([k], [v], path, _new(2, 1, dtype=torch.int32), 3, [kc], [vc])),
        (ValueError, "unit last-dim", lambda: mta.tree_commit([k], [v], path, count, 3, [_new(2, 2, 64, 32).transpose(2, 3)], [vc])),
        (ValueError, "same shape", lambda: mta.tree_commit([k], [v], path, count, 3, [kc], [vc[:, :, :9]])),
        (RuntimeError, "dtype and device", lambda: mta.tree_commit([k], [v], path, count, 3, [kc.half()], [vc.half()])),
        (RuntimeError, "unsupported dtype", lambda: mta.tree_commit([k.float()], [v.float()], path, count, 3, [kc.float()], [vc.float()])),
    )


def topk_verify(mta):
    x, tok, par = _new(2, 5, 40), _new(2, 5, dtype=torch.int64), _new(2, 5, dtype=torch.int32)
    u, e = _new(2, 5, dtype=torch.float32), _new(2, 40, dtype=torch.float32)
    f = mta.ops.topk_verify
    return (
        (ValueError, "1 <= k <= vocab", lambda: f(x, tok, par, u, e, 0)),
        (ValueError, "1 <= k <= vocab", lambda: f(x, tok, par, u, e, 41)),
        (ValueError, "32768", lambda: f(_new(2, 5, 32769), tok, par, u, _new(2, 32769, dtype=torch.float32), 8)),
        (ValueError, "1 to 64 nodes", lambda: f(_new(2, 65, 40), tok, par, u, e, 8)),
        (ValueError, r"\[batch, nodes, vocab\]", lambda: f(x[0], tok, par, u, e, 8)),
        (ValueError, "tokens must be", lambda: f(x, tok.int(), par, u, e, 8)),
        (ValueError, "parents must be", lambda: f(x, tok, par.long(), u, e, 8)),
        (ValueError, "uniform must be", lambda: f(x, tok, par, u[:, :4], e, 8)),
        (ValueError, "noise must be", lambda: f(x, tok, par, u, e.double(), 8)),
        (ValueError, "shape of logits", lambda: f(x, tok, par, u, e, 8, draft_logits=x[:, :4])),
        (RuntimeError, "dtype and device", lambda: f(x, tok, par, u, e, 8, draft_logits=x.float())),
        (RuntimeError, "unsupported", lambda: f(x.double(), tok, par, u, e, 8)),
    )


def topk_distillation(mta):
    x, y, i = _new(2, 3, 40), _new(2, 3, 7, dtype=torch.float32), _new(2, 3, 7, dtype=torch.int64)
    f = mta.ops.topk_distillation
    return (
        (ValueError, "rows of logits", lambda: f(x, y[:1], i[:1])),
        (ValueError, "rows of logits", lambda: f(x, y[0], i[0])),
        (ValueError, "shape of teacher_logits", lambda: f(x, y, i[..., :6])),
        (ValueError, "integer tensor", lambda: f(x, y, y)),
        (ValueError, "1 to 1024", lambda: f(x, _new(2, 3, 1025), _new(2, 3, 1025, dtype=torch.int64))),
        (ValueError, "1 to 1024", lambda: f(x, y[..., :0], i[..., :0])),
        (ValueError, "temperature", lambda: f(x, y, i, temperature=0.0)),
        (ValueError, "temperature", lambda: f(x, y, i, temperature=math.nan)),
        (ValueError, "temperature", lambda: f(x, y, i, temperature=math.inf)),
        (RuntimeError, "unsupported", lambda: f(x.double(), y, i)),
        (RuntimeError, "unsupported", lambda: f(x, y.double(), i)),
    )
