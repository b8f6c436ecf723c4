"""GPU: the LSE of every form of general attention's forward, gradients through each of them, and
the registered operators that give both.

The LSE (base 2, -inf without a key) is what the backward recomputes probabilities from.  Which
form a call takes - one CTA, a cluster of CTAs or equal shares for a few rows, whole or split
keys for many - depends on its sizes; each is held to the 64-bit oracle's bounds.
"""
import ctypes
import math

import pytest
import torch

from fastflashattention_b200 import _lib, cross_attention, relative_attention
from fastflashattention_b200._general import bucket_borders
from oracle.general_oracle import FINE, HALF, PAIR, attend, bucket_of

pytestmark = pytest.mark.gpu

TOL = 5e-3


def rnd(gen, *shape, size=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * size).to(torch.bfloat16)


def inputs(B, Hq, Hkv, Sq, Sk, D, seed=0, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (rnd(gen, B, Hq, Sq, D, size=size), rnd(gen, B, Hkv, Sk, D), rnd(gen, B, Hkv, Sk, D), rnd(gen, B, Hq, Sq, D))


def table(H, buckets=32, seed=11):
    return rnd(torch.Generator(device="cuda").manual_seed(seed), buckets, H, size=2.0)


def step_lengths(B, Sk):
    """Lengths of a padded batch: the longest, none, one, and others between."""
    return torch.tensor([(Sk, 0, 1, Sk // 3, Sk - 5, Sk // 2)[b % 6] for b in range(B)], dtype=torch.int32, device="cuda")


def mask_args(bias=None, causal=False, lengths=None, offsets=0, distance=128):
    """The operators' <mask> arguments and the oracle's, of the same mask."""
    borders = list(bucket_borders(bias.shape[0] // (1 if causal else 2), distance)) if bias is not None else []
    tensor = isinstance(offsets, torch.Tensor)
    both = bias is not None and not causal
    op = (bias, lengths, offsets if tensor else None, 0 if tensor else offsets, borders, both, causal, None)
    return op, dict(bias=bias, causal=causal, both=both, lengths=lengths, offsets=offsets, max_distance=distance)


def inside(got, want, name, gate=TOL):
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape and torch.isfinite(got).all(), name
    assert ((got - value).abs() - bound).max() <= 0, f"{name}: {float(((got - value).abs() - bound).max())} over the bound"
    if gate is not None and value.norm() > 0:
        assert (got - value).norm() <= gate * value.norm(), name


def lse_inside(got, want):
    """-inf exactly where no key is seen, and everywhere else inside the oracle's bound."""
    value, bound = want
    none = value == -math.inf
    assert got.dtype == torch.float32 and got.shape == value.shape
    assert torch.equal(got == -math.inf, none)
    far = torch.where(none, 0.0, (got.double() - value).abs() - bound)
    assert not torch.isnan(far).any() and far.max() <= 0, f"LSE: {float(far.max())} over the bound"


def check(q, k, v, do, grads=True, **mask):
    """o and LSE of general_lse, and what general_backward makes of them."""
    ops = _lib.ops()
    op, oracle = mask_args(**mask)
    want = attend(q, k, v, do if grads else None, exact=False, **oracle)
    o, lo, lse = ops.general_lse(q, k, v, *op, False)
    assert lo.numel() == 0
    inside(o, want["o"], "o")
    lse_inside(lse, want["lse"])
    if grads:
        dq, dk, dv, db = ops.general_backward(q, k, v, o, None, do, lse, *op, True, True, False)
        assert db.numel() == 0
        for name, g in (("dq", dq), ("dk", dk), ("dv", dv)):
            inside(g, want[name], name)
    assert _lib.device_status() == (0, 0, 0, 0)


# ---- a few rows ---------------------------------------------------------------------------

@pytest.mark.parametrize("items, rows, Sk, D", [
    (297, 1, 300, 64), (160, 1, 300, 128),                                        # one CTA for each item
    (148, 1, 600, 64), (64, 1, 1100, 64), (32, 1, 2100, 64), (12, 1, 4200, 64),   # clusters of 2, 4, 8, 16 CTAs
    (148, 9, 300, 128), (64, 9, 600, 128), (32, 9, 1100, 128), (12, 9, 2100, 128),
])
def test_lse_of_clusters(items, rows, Sk, D):
    check(*inputs(1, items, items, rows, Sk, D))
    check(*inputs(items, 1, 1, rows, Sk, D), lengths=step_lengths(items, Sk))
    lens = step_lengths(items, Sk)  # sequences that are shorter than their new tokens, too
    check(*inputs(items, 1, 1, rows, Sk, D), bias=table(1), causal=True, lengths=lens, offsets=lens - rows)


@pytest.mark.parametrize("items, Sk, D", [(148, 300, 64), (74, 600, 64), (32, 1100, 128), (14, 1100, 128), (6, 1100, 64)])
def test_lse_of_clusters_with_32_rows(items, Sk, D):
    check(*inputs(1, 4 * items, items, 6, Sk, D))
    check(*inputs(1, 4 * items, items, 6, Sk, D), bias=table(4 * items), offsets=Sk - 6, causal=True)


@pytest.mark.parametrize("B, Hkv, G, Sq, Sk, D, ragged", [
    (2, 4, 8, 3, 20000, 128, False), (4, 4, 4, 8, 20000, 64, True), (10, 10, 3, 7, 6000, 128, False),  # 32 rows
    (1, 13, 1, 1, 50000, 128, False), (1, 13, 9, 1, 100000, 64, False), (11, 3, 1, 1, 20000, 128, True),  # 16 rows
])
def test_lse_of_shares(B, Hkv, G, Sq, Sk, D, ragged):
    q, k, v, do = inputs(B, G * Hkv, Hkv, Sq, Sk, D)
    lens = step_lengths(B, Sk) if ragged else None
    p = _lib.GenProblem(batch=B, q_heads=G * Hkv, kv_heads=Hkv, q_len=Sq, k_len=Sk, head_dim=D, scale=1.0)
    if ragged:
        p.key_lengths = lens.data_ptr()
    assert _lib.load().ffa_gen_fwd_workspace(ctypes.byref(p), 0) > 0  # room for the parts
    check(q, k, v, do, lengths=lens)
    check(q, k, v, do, bias=table(G * Hkv), causal=True, lengths=lens, offsets=lens - Sq if ragged else Sk - Sq)


@pytest.mark.parametrize("B, Hkv, G, Sq, Sk, D", [
    (1, 12, 1, 1, 4200, 64), (40, 8, 1, 1, 300, 64), (1, 13, 1, 2, 50000, 128), (2, 4, 8, 3, 20000, 64),
])
def test_gradients_through_a_few_rows(B, Hkv, G, Sq, Sk, D):
    """The public calls: keys and values that want gradients, and a table that does not."""
    q, k, v, do = inputs(B, G * Hkv, Hkv, Sq, Sk, D)
    lens = step_lengths(B, Sk) if B > 1 else None
    bias = table(G * Hkv)
    for frozen in (None, bias):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        if frozen is None:
            o = cross_attention(*leaves, key_lengths=lens, enable_gqa=G > 1)
            want = attend(q, k, v, do, lengths=lens)
        else:
            o = relative_attention(*leaves, frozen, key_lengths=lens, query_offset=Sk // 2, enable_gqa=G > 1)
            want = attend(q, k, v, do, bias=frozen, both=True, lengths=lens, offsets=Sk // 2, exact=False)
        inside(o, want["o"], "o")
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)):
            inside(g, want[name], name)


@pytest.mark.parametrize("B, Hkv, G, Sq, Sk, D", [(2, 4, 8, 3, 20000, 128), (1, 12, 1, 1, 4200, 64)])
def test_captured_steps_with_gradients(B, Hkv, G, Sq, Sk, D):
    """Shares with their early join, and clusters of 16, forward and backward in two graphs that are
    replayed in turn over lengths that change."""
    q, k, v, do = inputs(B, G * Hkv, Hkv, Sq, Sk, D)
    bias = table(G * Hkv)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def step(lens):
        a = cross_attention(*leaves, key_lengths=lens, enable_gqa=True)
        b = relative_attention(*leaves, bias, query_offset=5, key_lengths=lens, enable_gqa=True)
        return [a.detach(), b.detach(), *torch.autograd.grad(a, leaves, do), *torch.autograd.grad(b, leaves, do)]

    graphs = []
    for n in range(2):
        lens = torch.full((B,), Sk - 7 * n, dtype=torch.int32, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(lens)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(lens)
        graphs.append((graph, lens, out))
    for less in (0, 1000, Sk // 2):
        for graph, lens, _ in graphs:
            lens -= less
            graph.replay()
        torch.cuda.synchronize()
        for _, lens, out in graphs:
            for x, y in zip(out, step(lens)):
                assert torch.equal(x, y)


# ---- many rows ----------------------------------------------------------------------------

@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("Sq, Sk", [(100, 4000), (300, 300), (1000, 77), (130, 0)])
def test_lse_of_whole_and_split_keys(Sq, Sk, D):
    check(*inputs(2, 2, 1, Sq, Sk, D), grads=Sk > 0)
    if Sk:
        lens = torch.tensor([Sk // 3, 0], dtype=torch.int32, device="cuda")
        check(*inputs(2, 2, 1, Sq, Sk, D), lengths=lens)
        check(*inputs(2, 2, 1, Sq, Sk, D), bias=table(2), causal=True, offsets=-70)  # rows without a key


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq, Sk", [(100, 4000), (300, 300)])
def test_remainder_of_o(Sq, Sk, D):
    """o + o_lo is O to 16 bits, whole and split, and the LSE beside it is the same contract's."""
    q, k, v, _ = inputs(2, 2, 1, Sq, Sk, D)
    op, oracle = mask_args(bias=table(2))
    want = attend(q, k, v, exact=True, **oracle)
    value, bound = want["o"]
    weighed = (bound - 1e-7 - HALF * value.abs()) / (HALF + FINE)  # P |V|
    o, lo, lse = _lib.ops().general_lse(q, k, v, *op, True)
    # what rounding O to nearest leaves is at most half a step.  (o + lo need not round to o: a
    # remainder just below half a step rounds to half a step, and o + lo is then a tie.)
    assert (lo.double().abs() <= HALF * o.double().abs()).all()
    fine = PAIR * value.abs() + (PAIR + FINE) * weighed + 1e-7
    inside(o.double() + lo.double(), (value, fine), "o + o_lo", gate=None)
    lse_inside(lse, want["lse"])


@pytest.mark.parametrize("want_dq, want_dkdv, want_db", [(True, False, False), (False, True, False), (True, True, True),
                                                         (False, False, True), (True, False, True), (False, True, True)])
def test_backward_operator_gives_what_is_wanted(want_dq, want_dkdv, want_db):
    q, k, v, do = inputs(2, 4, 2, 150, 170, 64)
    op, oracle = mask_args(bias=table(4))
    # the remainder is read with dQ, which dbias comes with
    want = attend(q, k, v, do, exact=want_dq or want_db, **oracle)
    o, lo, lse = _lib.ops().general_lse(q, k, v, *op, True)
    got = _lib.ops().general_backward(q, k, v, o, lo, do, lse, *op, want_dq, want_dkdv, want_db)
    for name, g, wanted in zip(("dq", "dk", "dv", "dbias"), got, (want_dq or want_db, want_dkdv, want_dkdv, want_db)):
        if wanted:
            inside(g, want[name], name, gate=None if name == "dbias" else TOL)
        else:
            assert g.numel() == 0


# ---- the bias's gradient -------------------------------------------------------------------

@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D, seed", [(64, 1), (128, 0)])
def test_remainder_of_o_is_what_the_bias_gradient_needs(D, seed, causal):
    """dbias adds dS over whole rows, whose sum is 0, so an error of delta = O . dO, common to a
    row, stays where dS cancels.  Values with a common mean leave dS as it is and enlarge that
    error.  With the remainder dbias is off by its own rounding to bf16, at most 2^-8 of each
    entry and so of the norm, and little else; without it, or without the forward that
    computes it, by 1.9 to 40 % of the norm (the same inputs in 64 bits with O, or P and O,
    rounded to bf16).  5e-3 lies between them."""
    gen = torch.Generator().manual_seed(seed)
    one = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16)  # noqa: E731
    B, H, S = 1, 2, 1485
    q, k = (one(B, H, S, D).float() * D ** -0.5).to(torch.bfloat16).cuda(), one(B, H, S, D).cuda()
    v, do = (one(B, H, S, D).float() + 4).to(torch.bfloat16).cuda(), one(B, H, S, D).cuda()
    bias = (torch.randn(16, H, generator=gen) * 2).to(torch.bfloat16).cuda()
    op, oracle = mask_args(bias=bias, causal=causal, distance=64)
    op = (*op[:-1], 1.0)
    value = attend(q, k, v, do, scale=1.0, **oracle)["dbias"][0]

    def off(g):
        return float((g.double() - value).norm() / value.norm())

    leaf = bias.clone().requires_grad_(True)
    o = relative_attention(q, k, v, leaf, max_distance=64, is_causal=causal, scale=1.0)
    public = off(torch.autograd.grad(o, [leaf], do)[0])
    ops = _lib.ops()
    o, lo, lse = ops.general_lse(q, k, v, *op, True)
    with_lo = off(ops.general_backward(q, k, v, o, lo, do, lse, *op, True, False, True)[3])
    dropped = off(ops.general_backward(q, k, v, o, None, do, lse, *op, True, False, True)[3])
    o, _, lse = ops.general_lse(q, k, v, *op, False)
    plain = off(ops.general_backward(q, k, v, o, None, do, lse, *op, True, False, True)[3])
    print(f"dbias off by {public:.5f} {with_lo:.5f}, without the remainder {dropped:.5f} {plain:.5f}")
    assert public <= TOL and with_lo <= TOL
    assert dropped > TOL and plain > TOL


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B, H, S, D, buckets, distance", [
    (2, 3, 70, 64, 32, 128), (1, 4, 385, 64, 16, 64), (1, 2, 700, 128, 64, 256), (2, 2, 300, 96, 256, 1024),
    (1, 6, 513, 64, 128, 800),
])
def test_bias_gradient_as_a_whole(B, H, S, D, buckets, distance, causal):
    """The norm of dbias's error where errors of different rows are independent: the rounding of
    the result, and four times the root of the rows' squared errors.  (The bound of each value
    adds up worst cases, and a few per cent of error stay inside it.)"""
    q, k, v, do = inputs(B, H, H, S, S, D, size=D ** -0.5)
    bias = table(H, buckets)
    _, oracle = mask_args(bias=bias, causal=causal, distance=distance)
    value, _ = attend(q, k, v, do, scale=1.0, **oracle)["dbias"]
    leaf = bias.clone().requires_grad_(True)
    o = relative_attention(q, k, v, leaf, max_distance=distance, is_causal=causal, scale=1.0)
    (g,) = torch.autograd.grad(o, [leaf], do)
    # a row's error: 2^-12 (exponentials, 32-bit sums) of its terms in each bucket
    qd, kd, vd, dd = (t.double() for t in (q, k, v, do))
    r = torch.arange(S, device="cuda")[None, :] - torch.arange(S, device="cuda")[:, None]
    bucket = bucket_of(r, buckets, distance, not causal)
    s = qd @ kd.transpose(-1, -2) + bias.double()[bucket].permute(2, 0, 1)
    if causal:
        s = s.masked_fill(r > 0, -math.inf)
    p, dp = torch.softmax(s, -1), dd @ vd.transpose(-1, -2)
    terms = p * (dp.abs() + (p * dp).sum(-1, keepdim=True).abs())
    rows = torch.zeros(B, H, S, buckets, device="cuda", dtype=torch.float64)
    rows.scatter_add_(3, bucket.expand(B, H, S, S), terms)
    assert (g.double() - value).norm() <= HALF * value.norm() + 4 * FINE * rows.norm()

