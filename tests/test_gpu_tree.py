"""GPU tests of the drafted-tree operators against the 64-bit oracle.

The bounds count roundings.  h is half a step of the output type.  Attention:
the probabilities and their sum are rounded alike, so an output value is off by at
most h (sum p |v| + |o|) from them and h |o| from its own rounding; the fp32 scores
of D products are off by at most (D + 8) 2^-24 sum |q k| each, which moves a
probability by that share (and its normaliser by as much again); exp and the sums
add less than 2^-16.  RoPE: three fp32 roundings of the two products and h."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import tree_oracle as orc
from tests import tree_refusals as refusals

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda:0"


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def np64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def trees(kind, b, n, seed):
    """Parents [b, n]: chains, bushes, forests of several roots, or with padding in every way it can be written."""
    rng = np.random.default_rng(seed)
    out = np.full((b, n), -1)
    for i in range(b):
        for j in range(1, n):
            out[i, j] = j - 1 if kind == "chain" else rng.integers(-1 if kind != "bush" else 0, j)
        if kind == "padded":
            for j in range(n):
                r = rng.random()
                if r < 0.3:
                    out[i, j] = rng.choice([-2, -100, j, j + 1, 1 << 20])
    return out


def rope_tables(rows, d):
    f = torch.outer(torch.arange(rows, dtype=torch.float64), 1.0 / 10_000.0 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))
    return f.cos().float().view(1, 1, rows, d // 2), f.sin().float().view(1, 1, rows, d // 2)


def attention_inputs(b, hq, hkv, d, n, cap, dtype, seed, sigma=1.0):
    g = gen(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * sigma).to(dtype)  # noqa: E731
    # [B, N, H, D] projections, [B, H, N, D] views
    q, k, v = (r(b, n, h, d).transpose(1, 2) for h in (hq, hkv, hkv))
    return [q, k, v, r(b, hkv, cap, d), r(b, hkv, cap, d)]


def check_attention(out, q, k, v, kc, vc, lengths, parents, name="", steps=0):
    """steps: fp32 additions of a long sum, beyond those that the 2^-16 covers."""
    d, h = q.shape[-1], half_step(out.dtype)
    got = np64(out)
    q, k, v, kc, vc = (np64(x) for x in (q, k, v, kc, vc))
    for i, (n, par) in enumerate(zip(lengths, parents)):
        ref, mag, top = orc.tree_attention(q[i], k[i], v[i], kc[i], vc[i], int(n), list(par), 1 / math.sqrt(d))
        share = 2 * (d + 8) * 2.0 ** -24 * (top[..., None] + 1) + 2.0 ** -16 + steps * 2.0 ** -24
        bound = (h + share) * (mag + abs(ref)) + h * abs(ref) + 1e-30
        if out.dtype == FP16:
            bound = bound + 2.0 ** -25  # half a step among the subnormals
        worst = float((abs(got[i] - ref) / bound).max())
        assert worst <= 1.0, f"{name} sequence {i} (length {n}): error {worst:.2f} of its bound"


@pytest.mark.parametrize("cases", [refusals.tree_attention, refusals.tree_rope_and_commit, refusals.topk_verify,
                                   refusals.topk_distillation], ids=lambda f: f.__name__)
def test_refusals_before_any_launch(mta, cases):
    for err, match, call in cases(mta):
        with pytest.raises(err, match=match):
            call()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
CASES = [
    # dtype, (query, KV heads), D, nodes, capacity, lengths, trees
    (BF16, (4, 4), 32, 1, 0, [0], "bush"),                        # one node, no cache
    (BF16, (8, 2), 64, 5, 64, [0, 1, 31, 32, 33, 63, 64], "chain"),  # both sides of a 32-key tile
    (FP16, (8, 2), 64, 33, 100, [100, 0, 7], "bush"),             # two tiles of nodes
    (BF16, (14, 2), 64, 7, 130, [130, 64, 1], "forest"),          # seven heads a group
    (BF16, (16, 1), 32, 64, 300, [300, 299], "bush"),             # 1024 query rows a KV head
    (FP16, (2, 2), 128, 64, 80, [80, 3], "padded"),
    (BF16, (32, 8), 128, 24, 1500, [1500, 700], "bush"),          # several workgroups a row block
    (BF16, (6, 2), 128, 11, 700, [700, 64, 0], "padded"),
    (BF16, (4, 2), 32, 64, 2000, [1999, 2000, 5], "chain"),
    (FP16, (8, 2), 64, 16, 4000, [4000, 1, 2000], "padded"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{str(c[0])[6:]}-{c[1][0]}x{c[1][1]}-d{c[2]}-n{c[3]}-cap{c[4]}-{c[6]}")
def test_tree_attention_matches_the_oracle(mta, case):
    dtype, (hq, hkv), d, n, cap, lengths, kind = case
    b = len(lengths)
    cpu = attention_inputs(b, hq, hkv, d, n, cap, dtype, seed=n + cap)
    par = trees(kind, b, n, seed=n)
    q, k, v, kc, vc = (x.to(DEV) for x in cpu)
    parents, length = (torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV) for x in (par, lengths))
    out = mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=hq // hkv)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    check_attention(out, *cpu, lengths, par)
    assert torch.equal(out, mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=hq // hkv)), "the same call twice"
    # an int length, a length and a tree for all
    same = mta.tree_attention(q, k, v, kc, vc, lengths[0], parents[0], repeats=hq // hkv)
    check_attention(same, *cpu, [lengths[0]] * b, [par[0]] * b, "int length")
    one = mta.tree_attention(q, k, v, kc, vc, length[:1], parents[0], repeats=hq // hkv)
    check_attention(one, *cpu, [lengths[0]] * b, [par[0]] * b, "one length")


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("repeats,n", [(4, 16), (4, 27), (8, 21)], ids=["rows64", "rows108", "rows168"])
def test_more_heads_than_the_card_takes_at_once(mta, repeats, n, d):
    """132 KV heads of all sequences, so that a workgroup takes 64, 128 and 256 query rows on one key tile: lengths
    about its tiles' ends, and padding and unseen cache rows that hold anything."""
    b, hkv, cap, dtype = 33, 4, 300, FP16 if d == 64 else BF16
    cpu = attention_inputs(b, hkv * repeats, hkv, d, n, cap, dtype, seed=n + d)
    par = trees("padded", b, n, seed=d)
    edges = [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 299, 300]
    lengths = [edges[i % 16] for i in range(b)]
    q, k, v, kc, vc = (x.to(DEV) for x in cpu)
    parents, length = (torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV) for x in (par, lengths))
    out = mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=repeats)
    pick = list(range(16)) + [b - 1]
    check_attention(out[pick], *(x[pick] for x in cpu), [lengths[i] for i in pick], par[pick])
    assert torch.equal(out, mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=repeats)), "the same call twice"
    padding = torch.tensor([[u is None for u in orc.ancestors(list(p))] for p in par], device=DEV)
    assert bool(padding.any()) and (out.transpose(1, 2)[padding] == 0).all()
    for bad in (math.nan, -math.inf):
        for x in (q, k, v):
            x.transpose(1, 2)[padding] = bad
        for i, m in enumerate(lengths):
            kc[i, :, m:] = bad
            vc[i, :, m:] = bad
        assert torch.equal(mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=repeats), out), bad


@pytest.mark.parametrize("d,n,cap", [(128, 16, 8300), (128, 16, 65700), (128, 64, 131200),
                                     (64, 64, 6300), (64, 64, 49300), (32, 64, 393300)])
def test_many_rows_on_a_long_cache(mta, d, n, cap):
    """64 heads of one KV head on caches so long that a workgroup takes 64, 128 and 256 rows, its keys shared out."""
    g = torch.Generator(DEV).manual_seed(cap)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF16)  # noqa: E731
    q, k, v, kc, vc = r(1, 64, n, d), r(1, 1, n, d), r(1, 1, n, d), r(1, 1, cap, d), r(1, 1, cap, d)
    par = trees("forest", 1, n, 6)
    parents = torch.tensor(par, dtype=torch.int32, device=DEV)
    for length in (cap - 33, cap):
        out = mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=64)
        one = [0 if length == cap else 63]
        check_attention(out[:, one], q[:, one], k, v, kc, vc, [length], par, steps=cap / 16)


def test_one_node_is_decode_attention(mta):
    """A tree of one node equals decode_attention with the node's row in the cache, to both rounding bounds."""
    b, hq, hkv, d, cap = 3, 8, 2, 64, 200
    cpu = attention_inputs(b, hq, hkv, d, 1, cap, BF16, seed=5)
    q, k, v, kc, vc = (x.to(DEV) for x in cpu)
    out = mta.tree_attention(q, k, v, kc, vc, 150, torch.full((1,), -1, dtype=torch.int32, device=DEV), repeats=4)
    kc2, vc2 = kc.clone(), vc.clone()
    kc2[:, :, 150:151], vc2[:, :, 150:151] = k, v
    ref = mta.decode_attention(q, kc2, vc2, 151, repeats=4)
    for x in (out, ref):
        check_attention(x, *cpu, [150] * b, [[-1]] * b)


def test_large_scores_and_equal_scores(mta):
    """Scores of several hundred (the running maximum moves at many keys), and all scores equal."""
    for sigma, name in ((6.0, "large"), (0.0, "equal")):
        cpu = attention_inputs(2, 4, 2, 64, 9, 300, BF16, seed=8, sigma=sigma or 1.0)
        if not sigma:
            cpu[0] = torch.zeros_like(cpu[0])
        par = trees("bush", 2, 9, 1)
        out = mta.tree_attention(*(x.to(DEV) for x in cpu), 300, torch.tensor(par, dtype=torch.int32, device=DEV), repeats=2)
        check_attention(out, *cpu, [300, 300], par, name)


def test_what_is_not_seen_may_hold_anything(mta):
    """NaN and infinities behind the cached length and in padding's queries, keys and values change nothing."""
    b, hq, hkv, d, n, cap = 4, 8, 2, 64, 40, 256
    q, k, v, kc, vc = (x.to(DEV) for x in attention_inputs(b, hq, hkv, d, n, cap, BF16, seed=2))
    par = trees("padded", b, n, 9)
    par[3] = -2  # a sequence of padding alone
    lengths = [100, 0, 256, 31]
    parents, length = (torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV) for x in (par, lengths))
    out = mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=4)
    padding = torch.tensor([[u is None for u in orc.ancestors(list(p))] for p in par], device=DEV)
    assert bool(padding.any()) and bool((~padding).any())
    assert (out.transpose(1, 2)[padding] == 0).all() and (out[3] == 0).all()
    for bad in (math.nan, math.inf, -math.inf):
        for x in (q, k, v):
            x.transpose(1, 2)[padding] = bad
        for i, m in enumerate(lengths):
            kc[i, :, m:] = bad
            vc[i, :, m:] = bad
        got = mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=4)
        assert torch.equal(got, out), bad


@pytest.mark.parametrize("b,hkv,repeats,n,d,dtype", [
    (3, 2, 4, 40, 64, BF16), (2, 1, 2, 64, 128, FP16), (2, 2, 1, 33, 32, BF16),
    (33, 4, 4, 16, 64, BF16), (33, 4, 4, 27, 128, FP16), (33, 4, 8, 21, 64, FP16), (33, 4, 8, 21, 32, BF16)])
def test_values_that_are_no_numbers_reach_descendants_alone(mta, b, hkv, repeats, n, d, dtype):
    cap, length = 70, 45
    cpu = attention_inputs(b, hkv * repeats, hkv, d, n, cap, dtype, seed=n)
    par = trees("forest", b, n, 12)
    dev = [x.to(DEV) for x in cpu]
    parents = torch.tensor(par, dtype=torch.int32, device=DEV)
    clean = mta.tree_attention(*dev, length, parents, repeats=repeats)
    bad = [1, n // 2, n - 1]
    for x in (cpu[2], dev[2]):
        x[:, :, bad[0], 0] = math.inf
        x[:, 0, bad[1], d - 1] = math.nan
        x[:, :, bad[2], d // 2] = -math.inf
    out = mta.tree_attention(*dev, length, parents, repeats=repeats)
    seen = torch.tensor([[[m in up for m in bad] for up in orc.ancestors(list(q))] for q in par])  # [B, N, 3]
    same = ~seen.any(-1)
    assert bool(same.any()) and bool(seen.any())
    assert torch.equal(out.transpose(1, 2).cpu()[same], clean.transpose(1, 2).cpu()[same])
    h = half_step(dtype)
    for i in (0, b - 1):
        with np.errstate(invalid="ignore"):
            ref, mag, top = orc.tree_attention(*(np64(x[i]) for x in cpu), length, list(par[i]), 1 / math.sqrt(d))
        got, fine = np64(out[i]), np.isfinite(ref)
        assert (fine == np.isfinite(got)).all() and (np.isnan(ref) == np.isnan(got)).all()
        assert (np.sign(ref) == np.sign(got))[np.isinf(ref)].all()
        share = 2 * (d + 8) * 2.0 ** -24 * (top[..., None] + 1) + 2.0 ** -16
        bound = (h + share) * (np.where(fine, mag, 0) + abs(ref)) + h * abs(ref) + 2.0 ** -25
        assert (abs(got[fine] - ref[fine]) <= bound[fine]).all()
    for x in dev[:2]:  # and the same of queries and keys
        x[:, :, bad] = math.nan
    out = mta.tree_attention(*dev, length, parents, repeats=repeats)
    assert torch.equal(out.transpose(1, 2).cpu()[same], clean.transpose(1, 2).cpu()[same])


def test_layouts_streams_and_clamped_lengths(mta):
    b, hq, hkv, d, n, cap = 2, 8, 2, 64, 12, 96
    cpu = attention_inputs(b, hq, hkv, d, n, cap, FP16, seed=4)
    par = trees("bush", b, n, 3)
    q, k, v, kc, vc = (x.to(DEV) for x in cpu)
    parents = torch.tensor(par, dtype=torch.int32, device=DEV)
    length = torch.tensor([96, 50], dtype=torch.int32, device=DEV)
    ref = mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=4)
    # slices of larger buffers, [B, T, H, D] caches, bases off 16 bytes, a last stride of 2
    big = torch.zeros(b, hkv, cap + 5, d + 8, dtype=FP16, device=DEV)
    big[:, :, 2:cap + 2, :d] = kc
    vt = vc.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(q.numel() + 1, dtype=FP16, device=DEV)[1:].view(b, hq, n, d).copy_(q)
    wide = torch.zeros(b, hkv, n, 2 * d, dtype=FP16, device=DEV)[..., ::2].copy_(k)
    got = mta.tree_attention(odd, wide, v.contiguous(), big[:, :, 2:cap + 2, :d], vt, length.flip(0).flip(0),
                             parents.t().contiguous().t(), repeats=4)
    assert torch.equal(got, ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    # lengths on the device are clamped to [0, capacity]
    far = torch.tensor([1 << 30, -7], dtype=torch.int32, device=DEV)
    check_attention(mta.tree_attention(q, k, v, kc, vc, far, parents, repeats=4), *cpu, [96, 0], par)


def test_offsets_past_32_bits(mta):
    """A cache of more than 2^32 bytes and 2^31 values: the last sequence's last position is the one that counts."""
    b, hkv, cap, d, n = 2, 9, 1_000_003, 128, 3
    kc = torch.zeros(b, hkv, cap, d, dtype=BF16, device=DEV)
    vc = torch.zeros_like(kc)
    assert kc.numel() > 1 << 31
    q, k, v = (torch.zeros(b, hkv, n, d, dtype=BF16, device=DEV) for _ in range(3))
    q[1, 8] = 8.0
    kc[1, 8, cap - 1] = 8.0  # its score is 8 * 8 * sqrt(128) = 724, every other 0
    vc[1, 8, cap - 1] = torch.arange(d, device=DEV).to(BF16)
    vc[0, 0, 0] = 1.0
    out = mta.tree_attention(q, k, v, kc, vc, cap, torch.tensor([-1, 0, 0], dtype=torch.int32, device=DEV), repeats=1)
    assert torch.equal(out[1, 8], vc[1, 8, cap - 1].expand(n, d))
    rest = torch.zeros_like(out)
    rest[1, 8] = out[1, 8]
    # sequence 0, head 0: the mean of one 1 and a million zeros and its own nodes'
    seen = torch.tensor([cap + 1, cap + 2, cap + 2], device=DEV, dtype=torch.float64)[:, None]
    assert ((out[0, 0].double() - 1 / seen).abs() <= 2 * half_step(BF16) / seen).all()
    rest[0, 0] = out[0, 0]
    assert torch.equal(out, rest)


def test_a_captured_step_follows_its_inputs(mta):
    """Rotation, attention, verification and commit recorded once; replays with other lengths, trees and numbers give
    the eager results, with eager work between them.  A second recording lives beside the first."""
    b, hq, hkv, d, n, cap, vocab = 3, 8, 2, 64, 8, 128, 500
    cos, sin = (t.to(DEV) for t in rope_tables(cap, d))
    g = gen(11)

    def inputs():
        q, k, v, kc, vc = (x.to(DEV) for x in attention_inputs(b, hq, hkv, d, n, cap, BF16, seed=int(torch.randint(1000, (1,), generator=g))))
        seed = int(torch.randint(1000, (1,), generator=g))
        return dict(q=q, k=k, v=v, kc=kc, vc=vc, length=torch.randint(0, cap - n, (b,), generator=g, dtype=torch.int32).to(DEV),
                    parents=torch.tensor(trees("bush", b, n, seed), dtype=torch.int32, device=DEV),
                    logits=torch.randn(b, n, vocab, generator=g).to(DEV), tokens=torch.randint(vocab, (b, n), generator=g).to(DEV),
                    uniform=torch.rand(b, n, generator=g).to(DEV) * 0.01, noise=torch.empty(b, vocab).exponential_(generator=g).to(DEV))

    def step(s):
        q, k = mta.tree_rope(s["q"], s["k"], cos, sin, s["length"], s["parents"])
        out = mta.tree_attention(q, k, s["v"], s["kc"], s["vc"], s["length"], s["parents"], repeats=4)
        path, count, token = mta.ops.topk_verify(s["logits"], s["tokens"], s["parents"], s["uniform"], s["noise"], 16)
        mta.tree_commit([k], [s["v"]], path, count, s["length"], [s["kc"]], [s["vc"]])
        return out, path, count, token, s["kc"], s["vc"]

    recorded = []
    for _ in range(2):
        static = inputs()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(static)
        recorded.append((graph, static, outs))
    for _ in range(3):
        for graph, static, outs in recorded:
            fresh = inputs()
            for name, x in fresh.items():
                static[name].copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            for got, ref in zip(outs, step(fresh)):
                assert torch.equal(got, ref)


# ---------------------------------------------------------------------------
# RoPE
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
@pytest.mark.parametrize("d,n,kind", [(32, 1, "chain"), (64, 64, "chain"), (128, 23, "padded"), (8, 64, "forest"), (72, 9, "bush")])
def test_tree_rope_matches_the_oracle(mta, dtype, d, n, kind):
    b, hq, hkv, rows = 3, 6, 2, 90
    q, k = attention_inputs(b, hq, hkv, d, n, 0, dtype, seed=d + n)[:2]
    cos, sin = rope_tables(rows, d)
    par, lengths = trees(kind, b, n, 7), [0, 89, 20]  # the second's deeper nodes take the last row
    got = mta.tree_rope(q.to(DEV), k.to(DEV), cos.to(DEV), sin.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV),
                        torch.tensor(par, dtype=torch.int32, device=DEV))
    for x, y in zip((q, k), got):
        assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
        for i in range(b):
            ref, mag = orc.tree_rope(np64(x[i]), np64(cos[0, 0]), np64(sin[0, 0]), lengths[i], list(par[i]))
            bound = half_step(dtype) * abs(ref) + 4 * 2.0 ** -24 * mag + 2.0 ** -25
            assert (abs(np64(y[i]) - ref) <= bound).all()
    ints = mta.tree_rope(q.to(DEV), k.to(DEV), cos.to(DEV), sin.to(DEV), 20, torch.tensor(par, dtype=torch.int32, device=DEV))
    assert all(torch.equal(x[2], y[2]) for x, y in zip(ints, got))
    # 16-bit tables off 16 bytes are read as the fp32 values they hold
    odd = [torch.zeros(t.numel() + 1, dtype=BF16, device=DEV)[1:].view(t.shape).copy_(t) for t in (cos, sin)]
    a = mta.tree_rope(q.to(DEV), k.to(DEV), *odd, 20, torch.tensor(par, dtype=torch.int32, device=DEV))
    e = mta.tree_rope(q.to(DEV), k.to(DEV), *(t.float().contiguous() for t in odd), 20, torch.tensor(par, dtype=torch.int32, device=DEV))
    assert all(torch.equal(x, y) for x, y in zip(a, e))


# ---------------------------------------------------------------------------
# the write into the caches
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("layers,d,dtype,layout", [(1, 64, BF16, "plain"), (35, 32, FP16, "plain"), (3, 36, BF16, "plain"),
                                                   (4, 64, BF16, "mixed")])
def test_tree_commit_writes_the_accepted_rows_alone(mta, layers, d, dtype, layout):
    b, hkv, n, cap = 4, 3, 9, 40
    g = gen(layers)
    path = torch.full((b, n), -1, dtype=torch.int32)
    path[0, :3] = torch.tensor([0, 2, 8])
    path[1, :9] = torch.arange(9)
    path[2, :4] = torch.tensor([0, 9, 3, -5])  # a node outside the tree and a negative one: skipped
    count, lengths = torch.tensor([3, 9, 4, 0], dtype=torch.int32), [5, 35, 0, 12]  # the second runs into the capacity
    make = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    nodes = [[make(b, n, hkv, d).to(DEV).transpose(1, 2) for _ in range(layers)] for _ in range(2)]
    caches = [[make(b, hkv, cap, d).to(DEV) for _ in range(layers)] for _ in range(2)]
    if layout == "mixed":  # other strides from layer to layer, a base off 16 bytes, a last stride of 2 among the nodes
        caches[0][1] = torch.empty(b, cap, hkv, d, dtype=dtype, device=DEV).copy_(caches[0][1].transpose(1, 2)).transpose(1, 2)
        caches[1][2] = torch.empty(b * hkv * cap * d + 1, dtype=dtype, device=DEV)[1:].view(b, hkv, cap, d).copy_(caches[1][2])
        nodes[0][3] = torch.empty(b, hkv, n, 2 * d, dtype=dtype, device=DEV)[..., ::2].copy_(nodes[0][3])
    want = [[c.clone() for c in cs] for cs in caches]
    for ns, ws in zip(nodes, want):
        for x, w in zip(ns, ws):
            for i in range(b):
                for j in range(int(count[i])):
                    node, pos = int(path[i, j]), lengths[i] + j
                    if 0 <= node < n and pos < cap:
                        w[i, :, pos] = x[i, :, node]
    mta.tree_commit(*nodes, path.to(DEV), count.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), *caches)
    for cs, ws in zip(caches, want):
        for c, w in zip(cs, ws):
            assert torch.equal(c, w)
    # counts past the nodes stop at them; an int length
    mta.tree_commit(*nodes, path.to(DEV), torch.full((b,), 1000, dtype=torch.int32, device=DEV), 4, *caches)
    assert torch.equal(caches[0][0][1, :, 4:13], nodes[0][0][1])


def test_tree_commit_refuses_shared_memory(mta):
    """Nodes that lie in a cache, and a cache that two layers would write; what only lies in one allocation is written."""
    g = gen(3)
    both = torch.randn(4, 2, 2, 40, 64, generator=g).to(BF16).to(DEV)  # two layers' key and value caches
    k, v = (torch.randn(2, 2, 5, 64, generator=g).to(BF16).to(DEV) for _ in range(2))
    path = torch.tensor([[0, 1, 3, -1, -1]] * 2, dtype=torch.int32, device=DEV)
    count = torch.full((2,), 3, dtype=torch.int32, device=DEV)
    before = both.clone()
    for keys, caches in (([both[0][:, :, 10:15]], [both[0]]), ([both[2][:, :, 10:15]], [both[0]]), ([k, v], [both[0], both[0]])):
        with pytest.raises(ValueError, match="overlap|take the nodes of two"):
            mta.tree_commit(keys, [v] * len(keys), path, count, 10, caches, [both[2], both[3]][:len(keys)])
    assert torch.equal(both, before)
    mta.tree_commit([k, k], [v, v], path, count, 10, [both[0], both[1]], [both[2], both[3]])
    for i, x in enumerate((k, k, v, v)):
        assert torch.equal(both[i][:, :, 10:13], x[:, :, [0, 1, 3]])
        assert torch.equal(both[i][:, :, 13:], before[i][:, :, 13:]) and torch.equal(both[i][:, :, :10], before[i][:, :, :10])


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------
def verify_inputs(b, n, vocab, k, dtype, drafted, seed, kind="bush"):
    g = gen(seed)
    x = (torch.randn(b, n, vocab, generator=g) * 2).to(dtype)
    y = (x.float() + torch.randn(b, n, vocab, generator=g)).to(dtype) if drafted else None
    par = trees(kind, b, n, seed)
    tokens = torch.zeros(b, n, dtype=torch.int64)
    for i in range(b):
        for j in range(n):
            u = par[i, j] if 0 <= par[i, j] < j else 0
            w = torch.from_numpy(orc.top_softmax(np64((y if drafted else x)[i, u]), k))
            tokens[i, j] = torch.multinomial(w, 1, generator=g)
    return dict(logits=x, tokens=tokens, parents=torch.tensor(par, dtype=torch.int32), uniform=torch.rand(b, n, generator=g),
                noise=torch.empty(b, vocab).exponential_(generator=g), k=k, draft_logits=y)


def check_verify(mta, s, name=""):
    path, count, token = mta.ops.topk_verify(**{a: x.to(DEV) if torch.is_tensor(x) else x for a, x in s.items()})
    b, n = s["tokens"].shape
    assert path.shape == (b, n) and count.shape == (b,) and token.shape == (b, 1)
    for i in range(b):
        par = s["parents"][i] if s["parents"].ndim == 2 else s["parents"]
        ref, drawn = orc.topk_verify(np64(s["logits"][i]), s["tokens"][i].tolist(), par.tolist(), np64(s["uniform"][i]),
                                     s["noise"][i].numpy(), s["k"], None if s["draft_logits"] is None else np64(s["draft_logits"][i]))
        assert path[i].tolist() == ref + [-1] * (n - len(ref)), f"{name} sequence {i}"
        assert int(count[i]) == len(ref) and int(token[i, 0]) == drawn, f"{name} sequence {i}"
    return path, count, token


@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("b,n,vocab,k,dtype,kind", [
    (8, 5, 300, 16, F32, "bush"),
    (4, 64, 1385, 50, BF16, "bush"),
    (4, 12, 8193, 1, F32, "bush"),
    (3, 9, 16384, 16, F32, "chain"),
    (2, 6, 32768, 16, FP16, "bush"),
    (3, 10, 2000, 1024, F32, "bush"),   # the largest k that keeps a list
    (3, 10, 2000, 1025, F32, "bush"),   # and past it
    (3, 10, 1100, 1100, F32, "bush"),   # every word kept
    (3, 7, 1, 1, F32, "bush"),
    (6, 9, 40, 8, F32, "padded"),
])
def test_topk_verify_matches_the_oracle(mta, b, n, vocab, k, dtype, kind, drafted):
    for seed in (1, 2):
        check_verify(mta, verify_inputs(b, n, vocab, k, dtype, drafted, seed, kind), f"seed {seed}")


@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("b,n,vocab,k,dtype,kind", [
    (40, 40, 300, 16, F32, "chain"),    # walks past the rows that are taken ahead
    (300, 9, 700, 4, BF16, "bush"),     # more sequences than the card takes at once
    (64, 24, 17001, 20, FP16, "bush"),
    (2, 6, 9000, 256, F32, "bush"),     # k at a workgroup's threads and past them, for each of its sizes
    (2, 6, 9000, 257, F32, "bush"),
    (2, 6, 20001, 512, F32, "bush"),
    (2, 6, 20001, 513, BF16, "bush"),
    (2, 6, 32768, 32768, F32, "bush"),
])
def test_topk_verify_past_the_card(mta, b, n, vocab, k, dtype, kind, drafted):
    check_verify(mta, verify_inputs(b, n, vocab, k, dtype, drafted, 5, kind))


def test_one_node_is_topk_sample(mta):
    for vocab, k in ((16384, 16), (1385, 50), (700, 700)):
        g = torch.Generator(device=DEV).manual_seed(vocab)
        x = torch.randn(9, 1, vocab, device=DEV, generator=g) * 3
        e = torch.empty(9, vocab, device=DEV).exponential_(generator=g)
        zero = torch.zeros(9, 1, dtype=torch.int64, device=DEV)
        path, count, token = mta.ops.topk_verify(x, zero, torch.full((1,), -1, dtype=torch.int32, device=DEV), zero.float(), e, k)
        assert torch.equal(token, mta.ops.topk_sample(x[:, 0], e, k)) and (count == 1).all() and (path == 0).all()


@pytest.mark.parametrize("drafted", [True, False])
def test_verify_ties_masks_and_odd_tokens(mta, drafted):
    """Whole-number logits (ties at the k-th value, more of them than a list holds), masked words of every kind, tokens
    outside the vocabulary, and siblings with the same token."""
    s = verify_inputs(6, 8, 3000, 5, F32, drafted, 4)
    s["logits"] = s["logits"].round().clamp(-1, 1)
    check_verify(mta, s, "ties")
    s = verify_inputs(6, 8, 64, 5, F32, drafted, 5)
    for j, bad in enumerate((-math.inf, math.nan, torch.finfo(F32).min)):
        s["logits"][2 * j:2 * j + 2, :, 3:] = bad  # fewer words left than k
    check_verify(mta, s, "masks")
    s["logits"][0] = -math.inf  # no word left: all alike
    s["logits"][1, :, 7] = math.inf
    check_verify(mta, s, "rows without a finite logit")
    s = verify_inputs(4, 8, 64, 5, F32, drafted, 6)
    s["parents"][:] = torch.tensor([-1, 0, 0, 0, 0, 0, 0, 0])
    s["tokens"][0] = s["tokens"][0, 1]
    s["tokens"][1] = torch.tensor([0, -1, 64, 1 << 40, -(1 << 40), 0, 1, 2])
    s["uniform"][:2] = 0.9
    check_verify(mta, s, "tokens")
    s["uniform"][:] = 0.0  # everything with a positive probability is taken
    check_verify(mta, s, "zeros")


@pytest.mark.parametrize("vocab", [40, 5000, 20000])
def test_verify_counts_infinity_as_the_highest_number(mta, vocab):
    # +inf and the largest float are one logit: with k = 1 both words stay, and the noise decides
    for k, at in ((1, 4), (1, vocab - 1), (2, vocab - 1)):
        s = verify_inputs(3, 2, vocab, k, F32, False, vocab + k)
        s["logits"][:, :, 3] = math.inf
        s["logits"][:, :, at] = torch.finfo(F32).max
        s["tokens"][:, 1] = at
        s["uniform"][:] = torch.tensor([[0.0, 0.25], [0.0, 0.75], [0.0, 0.75]])
        s["noise"][:, 3] = 2.0
        s["noise"][1, 3], s["noise"][0, at], s["noise"][2, at] = 3.0, 1.0, 4.0
        path, count, token = check_verify(mta, s, f"k {k} at {at}")
        assert count.tolist() == [2, 1, 1] and token.flatten().tolist() == [at, 3, 3]


def test_verify_layouts(mta):
    s = verify_inputs(4, 6, 515, 16, BF16, True, 7)
    dev = {a: x.to(DEV) if torch.is_tensor(x) else x for a, x in s.items()}
    ref = mta.ops.topk_verify(**dev)
    wide = torch.zeros(6, 4, 600, dtype=BF16, device=DEV)
    wide[:, :, 1:516] = dev["logits"].transpose(0, 1)
    dev["logits"] = wide[:, :, 1:516].transpose(0, 1)  # rows off 16 bytes, nodes outermost
    dev["noise"] = torch.zeros(4, 700, device=DEV)[:, 3:518].copy_(dev["noise"])
    dev["tokens"] = dev["tokens"].t().contiguous().t()
    dev["draft_logits"] = torch.zeros(4, 6, 1030, dtype=BF16, device=DEV)[..., ::2].copy_(dev["draft_logits"])
    for a, e in zip(mta.ops.topk_verify(**dev), ref):
        assert torch.equal(a, e)
    one = dict(s, parents=s["parents"][0])
    check_verify(mta, one, "one tree for all")
    none = mta.ops.topk_verify(dev["logits"][:0], dev["tokens"][:0], s["parents"][0].to(DEV), dev["uniform"][:0], dev["noise"][:0], 16)
    assert [tuple(t.shape) for t in none] == [(0, 6), (0,), (0, 1)]


def test_verify_frequencies(mta):
    """16384 walks over one tree: the token after node 0 follows the target's top-k softmax, within 5 standard deviations."""
    b, v, k = 16384, 12, 6
    g = torch.Generator(device=DEV).manual_seed(0)
    x, y = torch.randn(4, v, device=DEV, generator=g) * 1.5, torch.randn(4, v, device=DEV, generator=g) * 1.5
    q = torch.from_numpy(orc.top_softmax(np64(y[0]), k)).to(DEV)
    tokens = torch.multinomial(q.expand(b, v), 4, replacement=True, generator=g)
    path, count, token = mta.ops.topk_verify(
        x.expand(b, 4, v), tokens, torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device=DEV),
        torch.rand(b, 4, device=DEV, generator=g), torch.empty(b, v, device=DEV).exponential_(generator=g), k,
        draft_logits=y.expand(b, 4, v))
    first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], token[:, 0])
    seen, p = np.bincount(first.cpu().numpy(), minlength=v), orc.top_softmax(np64(x[0]), k)
    assert (abs(seen - b * p) <= 5 * np.sqrt(b * p * (1 - p)) + 1e-9).all()
    assert 0 < int((count > 1).sum()) < b


# ---------------------------------------------------------------------------
# the operators together, as a model generates with them
# ---------------------------------------------------------------------------
def test_a_model_generates_with_drafted_trees(mta):
    """A decoder that feeds drafted trees, verifies them with k = 1 (the target's likeliest word) and commits the
    accepted nodes: every token it emits is the full forward's likeliest for the text before it, up to the 16-bit
    caches (the same gap that the one-token decode is allowed), and good drafts are accepted."""
    torch.manual_seed(0)
    model = mta.model.TradingModel(61, 64, hidden_dim=128, layers=2, attention_heads=4, kv_heads=2, dropout=0.0,
                                   attention_backend="hip").to(DEV).eval()
    with torch.no_grad():
        for p in model.parameters():
            p.mul_(3.0)
    d, b = 32, 2
    parents = torch.tensor([-1, 0, 0, 1, 3], dtype=torch.int32, device=DEV)

    @torch.no_grad()
    def tree_pass(tokens, caches, length):
        """Logits [B, N, vocab] after every node, and the nodes' keys and values of every layer."""
        hidden, ks, vs = model.token_embedding(tokens), [], []
        for block, (kc, vc) in zip(model.blocks, caches):
            q, k, v = (x.to(BF16) for x in block.attention._heads(block.attention_norm(hidden)))
            q, k = mta.tree_rope(q, k, block.attention.rope.cos, block.attention.rope.sin, length, parents)
            a = mta.tree_attention(q, k, v, kc, vc, length, parents, repeats=2).float()
            hidden = hidden + block.attention._out(a.transpose(1, 2).reshape(hidden.shape))
            hidden = hidden + block.feed_forward(block.ffn_norm(hidden))
            ks.append(k)
            vs.append(v)
        return model.output(model.norm(hidden)), ks, vs

    text = [row.tolist() for row in torch.randint(61, (b, 7), device=DEV)]
    start = torch.tensor(text, device=DEV)
    with torch.no_grad():
        _, caches, _ = model._prefill(start[:, :-1])
    length = torch.full((b,), 6, dtype=torch.int32, device=DEV)
    last = start[:, -1:]
    accepted = 0
    g = torch.Generator(device=DEV).manual_seed(1)
    for step in range(6):
        # drafts: in every other step the model's own likeliest words, else anything
        tokens = torch.randint(61, (b, 5), device=DEV, generator=g)
        tokens[:, :1] = last
        if step % 2:
            for i, row in enumerate(text):
                ahead = list(row)
                for node in (1, 3):
                    with torch.no_grad():
                        ahead.append(int(model(torch.tensor([ahead], device=DEV))[0, -1].argmax()))
                    tokens[i, node] = ahead[-1]
        logits, ks, vs = tree_pass(tokens, caches, length)
        noise = torch.empty(b, 61, device=DEV).exponential_(generator=g)
        path, count, token = mta.ops.topk_verify(logits, tokens, parents, torch.rand(b, 5, device=DEV, generator=g), noise, 1)
        mta.tree_commit(ks, vs, path, count, length, [c[0] for c in caches], [c[1] for c in caches])
        length += count
        last = token
        for i, row in enumerate(text):
            new = [int(tokens[i, n]) for n in path[i, 1:int(count[i])].tolist()] + [int(token[i, 0])]
            accepted += len(new) - 1
            for x in new:
                with torch.no_grad():
                    full = model(torch.tensor([row], device=DEV))[0, -1]
                assert float(full.max() - full[x]) <= 2e-2 * float(full.abs().max()), (step, i)
                row.append(x)
            assert int(length[i]) == len(row) - 1
    assert accepted >= 6
