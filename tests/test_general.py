"""GPU: cross_attention and relative_attention against the definition in 64 bits.

Every value of every output is held to the bound that the oracle derives from the documented
roundings (oracle/general_oracle.py), and every output to the package's gate of 5e-3
relative L2 (typical errors are far below the bound, which adds up worst cases).
"""
import ctypes
import math
import threading

import pytest
import torch
from torch.autograd import forward_ad

from fastflashattention_b200 import (RelativeFlashAttention, UnsupportedConfig, _lib, cross_attention, fast_attention,
                                     relative_attention)
from fastflashattention_b200._general import bucket_borders
from oracle.general_oracle import attend

pytestmark = pytest.mark.gpu

TOL = 5e-3


def rnd(gen, *shape, size=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * size).to(torch.bfloat16)


def inputs(B, Hq, Hkv, Sq, Sk, D, layout="bhsd", seed=0, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    def one(H, S, size=1.0):
        if layout == "bshd":
            return rnd(gen, B, S, H, D, size=size).transpose(1, 2)
        return rnd(gen, B, H, S, D, size=size)
    return one(Hq, Sq, size), one(Hkv, Sk), one(Hkv, Sk), one(Hq, Sq)


def near(got, want, name, gate=TOL):
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, name
    assert torch.isfinite(got).all(), name
    far = (got - value).abs() - bound
    assert far.max() <= 0, f"{name}: {float(far.max())} over the bound at {int(far.argmax())}"
    norm = value.norm()
    # The gate is for sums that do not cancel.  A row's dS adds up to 0, so where a bucket
    # holds most of a row its share of dbias is small beside its terms (0, where one bucket
    # holds all): there the error may be what the oracle derives for those terms.
    free = (bound - 2.0 ** -8 * value.abs()).norm() if name == "dbias" else 0.0
    if norm > 0:  # else the bound says all: one key, whose dS is 0
        assert (got - value).norm() <= gate * norm + free, f"{name}: rel L2 {float((got - value).norm() / norm)}"


def check(q, k, v, do, bias=None, train=True, gate=TOL, **kw):
    """Forward and gradients of the public call against the oracle."""
    oracle_kw = dict(scale=kw.get("scale"), lengths=kw.get("key_lengths"))
    if bias is not None:
        oracle_kw.update(bias=bias, max_distance=kw.get("max_distance", 128), causal=kw.get("is_causal", False),
                         both=kw.get("bidirectional", not kw.get("is_causal", False)), offsets=kw.get("query_offset", 0))
    want = attend(q, k, v, do if train else None, **oracle_kw)
    gqa = q.shape[1] != k.shape[1]
    call = lambda q, k, v, b: (cross_attention(q, k, v, enable_gqa=gqa, **kw) if b is None else  # noqa: E731
                               relative_attention(q, k, v, b, enable_gqa=gqa, **kw))
    near(call(q, k, v, bias), want["o"], "o", gate)
    if train:
        leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for t in (q, k, v)]
        b = bias.detach().clone().requires_grad_(True) if bias is not None else None
        o = call(*leaves, b)
        near(o, want["o"], "o with gradients", gate)
        grads = torch.autograd.grad(o, leaves + ([b] if b is not None else []), do)
        for name, g in zip(("dq", "dk", "dv", "dbias"), grads):
            assert g.dtype == torch.bfloat16
            near(g, want[name], name, gate)
    assert _lib.device_status() == (0, 0, 0, 0)
    return want


# ---- cross attention -------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
@pytest.mark.parametrize("B, Hq, Hkv, Sq, Sk, D", [
    (1, 1, 1, 1, 1, 64), (2, 3, 3, 1, 77, 64), (1, 2, 1, 127, 129, 64), (2, 4, 2, 130, 63, 64), (1, 2, 2, 65, 300, 32),
    (2, 2, 2, 100, 200, 8), (1, 4, 1, 257, 65, 40), (1, 2, 2, 300, 513, 128), (2, 6, 2, 129, 127, 96),
    (1, 2, 2, 256, 256, 80), (1, 8, 1, 20, 700, 128), (1, 1, 1, 1000, 1, 64), (1, 1, 1, 1, 1000, 128),
])
def test_cross(B, Hq, Hkv, Sq, Sk, D, layout):
    check(*inputs(B, Hq, Hkv, Sq, Sk, D, layout))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 3, 70, 200])
def test_cross_key_lengths(D, Sq):
    """Lengths of zero, one, a tile's border and beyond; rows behind a length hold NaN."""
    lengths = [0, 1, 63, 64, 65, 127, 128, 129, 250, 300, 999, -7]
    q, k, v, do = inputs(len(lengths), 4, 2, Sq, 300, D, "bshd")
    for b, n in enumerate(lengths):
        k[b, :, max(0, min(n, 300)):] = math.nan
        v[b, :, max(0, min(n, 300)):] = math.nan
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = check(q, k, v, do, key_lengths=lens)
    assert (want["o"][0][0] == 0).all()
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    o = cross_attention(*leaves, key_lengths=lens, enable_gqa=True)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    assert (o[0] == 0).all() and (o[-1] == 0).all() and (dq[0] == 0).all()
    for b, n in enumerate(lengths):  # keys that nobody sees: exactly no gradient
        assert (dk[b, :, max(0, n):] == 0).all() and (dv[b, :, max(0, n):] == 0).all()


@pytest.mark.parametrize("G, Sq", [(1, 1), (8, 1), (9, 1), (16, 1), (3, 5), (17, 1), (8, 4), (11, 3), (16, 4), (1, 64),
                                   (1, 65), (13, 5)])
@pytest.mark.parametrize("D", [40, 128])
def test_few_rows(G, Sq, D):
    """Every way of putting the rows of a key head together, over keys that many CTAs share."""
    q, k, v, do = inputs(3, 2 * G, 2, Sq, 2500, D)
    check(q, k, v, do, train=False, key_lengths=torch.tensor([2500, 3, 1111], dtype=torch.int32, device="cuda"))
    check(q[:1], k[:1], v[:1], do[:1], train=False)


@pytest.mark.parametrize("B, Hkv, Sk", [(1, 1, 20000), (1, 3, 5000), (40, 4, 130), (5, 37, 300), (300, 1, 200)])
@pytest.mark.parametrize("D", [64, 96])
def test_few_rows_shares(B, Hkv, Sk, D):
    q, k, v, _ = inputs(B, Hkv, Hkv, 1, Sk, D)
    gen = torch.Generator(device="cuda").manual_seed(1)
    check(q, k, v, None, train=False)
    lens = torch.randint(0, Sk + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
    check(q, k, v, None, train=False, key_lengths=lens)


def step_lengths(B, Sk):
    """Lengths of a padded batch: the longest, none, one, and others between."""
    return torch.tensor([(Sk, 0, 1, Sk // 3, Sk - 5, Sk // 2)[b % 6] for b in range(B)], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("items", [12, 13, 32, 33, 64, 65, 148, 149, 296, 297])
@pytest.mark.parametrize("rows, D", [(1, 64), (9, 128)])
def test_clusters_of_ctas(items, rows, D):
    """As many items as clusters of 16, 8, 4, 2 and 1 CTAs fit at once, and one more."""
    Sk = 4200 if D == 64 else 2100
    q, k, v, _ = inputs(1, items, items, rows, Sk, D)
    check(q, k, v, None, train=False)
    q, k, v, _ = inputs(items, 1, 1, rows, Sk, D)
    check(q, k, v, None, train=False, key_lengths=step_lengths(items, Sk))


@pytest.mark.parametrize("items", [6, 14, 15, 32, 33, 74, 75, 148, 149])
@pytest.mark.parametrize("D", [64, 128])
def test_clusters_of_ctas_with_32_rows(items, D):
    q, k, v, _ = inputs(1, 4 * items, items, 6, 1500, D)
    check(q, k, v, None, train=False)
    check(q, k, v, None, table(32, 4 * items), train=False, is_causal=True, query_offset=1400)


@pytest.mark.parametrize("B, Hkv, G, Sq, Sk, D, ragged, shares", [
    (2, 4, 8, 3, 20000, 128, False, True), (4, 4, 4, 8, 20000, 64, True, True),  # 32 rows
    (10, 10, 3, 7, 2560, 128, False, False), (10, 10, 3, 7, 6000, 128, False, True),
    (1, 13, 1, 1, 50000, 128, False, True), (1, 13, 9, 1, 100000, 64, False, True),  # 16 rows
    (11, 3, 1, 1, 20000, 128, True, True),
])
def test_shares(B, Hkv, G, Sq, Sk, D, ragged, shares):
    """Equal shares of all keys, whose parts a second kernel joins (one shape that the estimate
    of time gives to single CTAs, 35.0 against 34.0)."""
    q, k, v, _ = inputs(B, G * Hkv, Hkv, Sq, Sk, D)
    lens = step_lengths(B, Sk) if ragged else None
    p = _lib.GenProblem(batch=B, q_heads=G * Hkv, kv_heads=Hkv, q_len=Sq, k_len=Sk, head_dim=D, scale=1.0)
    if ragged:
        p.key_lengths = lens.data_ptr()
    assert (_lib.load().ffa_gen_fwd_workspace(ctypes.byref(p), 0) > 0) == shares  # room for the parts
    check(q, k, v, None, train=False, key_lengths=lens)
    where = {"key_lengths": lens, "query_offset": lens - Sq} if ragged else {"query_offset": Sk - Sq}
    check(q, k, v, None, table(32, G * Hkv), train=False, is_causal=True, **where)


@pytest.mark.parametrize("Sq, Sk, D", [(100, 4000, 64), (100, 4000, 128), (4000, 100, 64), (4000, 100, 128)])
def test_split_and_joined(Sq, Sk, D):
    """Few CTAs over a long axis: keys (forward, dQ) and queries (dK, dV) are split and joined."""
    q, k, v, do = inputs(2, 2, 1, Sq, Sk, D, "bshd")
    check(q, k, v, do)
    check(q, k, v, do, key_lengths=torch.tensor([Sk // 3, Sk], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_scales(scale):
    check(*inputs(1, 2, 2, 150, 200, 64), scale=scale)
    check(*inputs(1, 2, 2, 2, 200, 64), scale=scale)
    check(*inputs(1, 2, 2, 300, 200, 128), scale=scale)


def test_large_scores():
    """Scores of several hundred (peaked softmax), and a max that grows late."""
    q, k, v, do = inputs(1, 2, 2, 200, 400, 64, size=8.0)
    k = k * torch.linspace(0.1, 4.0, 400, device="cuda").to(torch.bfloat16)[:, None]
    check(q, k, v, do, train=False)


def test_same_as_fast_attention_on_equal_shapes():
    q, k, v, do = inputs(2, 4, 4, 512, 512, 64)
    a, b = cross_attention(q, k, v), fast_attention(q, k, v)
    want = attend(q, k, v)["o"]
    near(a, want, "cross")
    near(b, want, "fast")


# ---- strides -----------------------------------------------------------------------------

def test_views_of_packed_projections():
    gen = torch.Generator(device="cuda").manual_seed(5)
    kv = rnd(gen, 2, 90, 2, 4, 64)  # [B, S, (k, v), H, D]
    qp = rnd(gen, 2, 70, 4, 64 + 16)  # a wider row
    q, k, v = qp[..., :64].transpose(1, 2), kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    check(q, k, v, rnd(gen, 2, 70, 4, 64).transpose(1, 2))
    check(q[:, :, ::3], k[:, :, ::2], v[:, :, ::2], rnd(gen, 2, 4, 24, 64))


def test_layouts_that_are_copied():
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k, v, do = inputs(2, 2, 2, 50, 60, 64)
    flat = rnd(gen, 2 * 2 * 60 * 64 + 3)
    odd = flat[3:].view(2, 2, 60, 64)  # off a 16-byte border
    check(q, odd, v, do)
    wide = rnd(gen, 2, 2, 60, 65)[..., :64]  # a row stride that is no multiple of 8
    check(q, k, wide, do)
    swapped = rnd(gen, 2, 2, 64, 60).transpose(2, 3)  # head dim not contiguous
    check(q, swapped, v, do)


def test_expanded_inputs_and_gradients():
    """Keys broadcast over the batch, and an output gradient of stride 0: gradients add up."""
    q, k, v, _ = inputs(3, 2, 2, 40, 50, 64)
    ke = k[:1].clone().requires_grad_(True)
    q2 = q.clone().requires_grad_(True)
    cross_attention(q2, ke.expand(3, -1, -1, -1), v).sum().backward()
    want = attend(q, k[:1].expand(3, -1, -1, -1), v, torch.ones_like(q))
    near(q2.grad, want["dq"], "dq")
    value, bound = want["dk"]
    # three bf16 gradients are added in bf16: two more roundings of partial sums
    near(ke.grad, (value.sum(0, keepdim=True), (bound + 2.0 ** -7 * value.abs()).sum(0, keepdim=True)), "dk", 1e-2)


def test_offsets_beyond_32_bits():
    """A cache of more than 2**31 elements: the last heads' keys lie behind that."""
    B, H, Sk, D = 2, 40, 440000, 64
    assert B * H * Sk * D > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(7)
    k, v = (torch.empty(B, H, Sk, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for t in (k, v):
        for b in range(B):
            t[b].copy_(torch.randn(H, Sk, D, device="cuda", generator=gen, dtype=torch.float32).to(torch.bfloat16))
    q = rnd(gen, B, H, 1, D)
    o = cross_attention(q, k, v)
    want = attend(q[-1:, -2:], k[-1:, -2:], v[-1:, -2:])["o"]
    near(o[-1:, -2:], want, "o")
    q = rnd(gen, 1, H, 130, D)
    o = cross_attention(q, k[1:], v[1:], key_lengths=torch.tensor([3000], dtype=torch.int32, device="cuda"))
    near(o[:, -1:], attend(q[:, -1:], k[1:, -1:, :3000], v[1:, -1:, :3000])["o"], "o of the last head")


@pytest.mark.parametrize("B, Hq, Hkv, Sq, Sk", [(0, 2, 2, 4, 5), (2, 0, 0, 4, 5), (2, 2, 2, 0, 5), (2, 2, 2, 4, 0),
                                                (2, 2, 2, 200, 0), (2, 2, 2, 0, 300)])
def test_empty(B, Hq, Hkv, Sq, Sk):
    q, k, v = (torch.randn(B, h, s, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)
               for h, s in ((Hq, Sq), (Hkv, Sk), (Hkv, Sk)))
    bias = torch.zeros(32, Hq, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    for o, leaves in ((cross_attention(q, k, v), (q, k, v)), (relative_attention(q, k, v, bias), (q, k, v, bias))):
        assert o.shape == (B, Hq, Sq, 64) and (o == 0).all()
        for g, t in zip(torch.autograd.grad(o, leaves, torch.ones_like(o)), leaves):
            assert g.shape == t.shape and (g == 0).all()


@pytest.mark.parametrize("Hkv", [0, 2])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [4, 300])
def test_no_query_heads(Hkv, Sq, D):
    """No query heads, over key heads too: an empty output, and zeros for every key and value."""
    q, k, v = (torch.randn(2, h, s, D, device="cuda").to(torch.bfloat16).requires_grad_(True)
               for h, s in ((0, Sq), (Hkv, 200), (Hkv, 200)))
    bias = torch.zeros(32, 0, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    calls = [(cross_attention(q, k, v, enable_gqa=True), (q, k, v))]
    for causal in (False, True):
        calls.append((relative_attention(q, k, v, bias, is_causal=causal, enable_gqa=True), (q, k, v, bias)))
    for o, leaves in calls:
        assert o.shape == (2, 0, Sq, D)
        for g, t in zip(torch.autograd.grad(o, leaves, torch.ones_like(o)), leaves):
            assert g.shape == t.shape and (g == 0).all()
    with torch.no_grad():
        assert relative_attention(q, k, v, bias, is_causal=True, enable_gqa=True).shape == (2, 0, Sq, D)
    assert _lib.device_status() == (0, 0, 0, 0)


# ---- relative position bias --------------------------------------------------------------

def table(buckets, H, seed=11, size=2.0):
    return rnd(torch.Generator(device="cuda").manual_seed(seed), buckets, H, size=size)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B, Hq, Hkv, S, D, buckets, distance", [
    (1, 1, 1, 1, 64, 32, 128), (2, 3, 3, 70, 64, 32, 128), (1, 2, 1, 127, 40, 32, 128), (1, 4, 2, 385, 64, 16, 64),
    (1, 2, 2, 700, 128, 64, 256), (2, 2, 1, 300, 96, 256, 1024), (1, 2, 2, 260, 128, 4, 3), (1, 6, 2, 513, 64, 128, 800),
])
def test_relative(B, Hq, Hkv, S, D, buckets, distance, causal):
    q, k, v, do = inputs(B, Hq, Hkv, S, S, D, "bshd", size=D ** -0.5)
    check(q, k, v, do, table(buckets, Hq), max_distance=distance, is_causal=causal, scale=1.0)


@pytest.mark.parametrize("D", [64, 128])
def test_relative_unidirectional_without_a_mask(D):
    q, k, v, do = inputs(1, 2, 2, 300, 300, D)
    check(q, k, v, do, table(32, 2), bidirectional=False)


@pytest.mark.parametrize("Sq", [1, 4, 100, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_new_tokens_over_a_cache(Sq, D):
    """The last Sq tokens of caches of different lengths; what lies behind is NaN."""
    lengths = [Sq, 333, 640, 700]
    q, k, v, do = inputs(4, 4, 2, Sq, 700, D)
    for b, n in enumerate(lengths):
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.nan
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    check(q, k, v, do, table(32, 4), is_causal=True, query_offset=lens - Sq, key_lengths=lens)
    # the mask alone keeps the rest of a cache out, too
    check(q, k, v, do, table(32, 4), is_causal=True, query_offset=lens - Sq)


@pytest.mark.parametrize("offset", [-1000, -150, -64, 37, 500, 2 ** 29])
@pytest.mark.parametrize("causal", [False, True])
def test_query_offsets(offset, causal):
    """Offsets that leave rows without a key, and positions far from any key."""
    q, k, v, do = inputs(1, 2, 2, 200, 260, 64)
    check(q, k, v, do, table(32, 2), is_causal=causal, query_offset=offset)
    check(q[:, :, :2], k, v, do[:, :, :2], table(32, 2), is_causal=causal, query_offset=offset)


def test_offsets_of_a_tensor_are_clamped():
    q, k, v, do = inputs(2, 2, 2, 100, 120, 64)
    far = torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    got = relative_attention(q, k, v, table(32, 2), query_offset=far)
    want = relative_attention(q, k, v, table(32, 2), query_offset=torch.tensor([2 ** 29, -2 ** 29], dtype=torch.int32,
                                                                              device="cuda"))
    assert torch.equal(got, want)


def test_masked_buckets():
    """A bucket of -inf hides its keys; rows that see nothing else are zero."""
    q, k, v, do = inputs(1, 2, 2, 300, 300, 64)
    bias = table(32, 2)
    bias[5] = -math.inf   # distance 5 behind
    bias[15] = -math.inf  # the last bucket behind: all far keys
    check(q, k, v, do, bias)
    check(q[:, :, :3], k, v, do[:, :, :3], bias)
    all_hidden = torch.full_like(bias, -math.inf)
    for n in (3, 300):
        assert (relative_attention(q[:, :, :n], k, v, all_hidden) == 0).all()


def test_lowest_values_act_as_documented():
    """Entries beyond 2**14 act as 2**14: the type's lowest value everywhere changes nothing."""
    q, k, v, do = inputs(1, 2, 2, 200, 200, 64)
    low = torch.full((32, 2), torch.finfo(torch.bfloat16).min, device="cuda", dtype=torch.bfloat16)
    plain = attend(q, k, v)["o"]
    # scores of a few units beside 2**14 * log2(e): their last place is 2**-9, of a probability too
    value, bound = plain
    for n in (2, 200):
        o = relative_attention(q[:, :, :n], k, v, low).double()
        assert ((o - value[:, :, :n]).abs() <= bound[:, :, :n] + 2.0 ** -8 * v.double().abs().amax()).all()
    one = table(32, 2)
    one[0] = torch.finfo(torch.bfloat16).min  # distance 0 alone: as good as hidden
    hidden = one.clone()
    hidden[0] = -math.inf
    assert torch.equal(relative_attention(q, k, v, one), relative_attention(q, k, v, hidden))


@pytest.mark.parametrize("n", [2, 200])
def test_entries_above_the_clamp_act_as_it(n):
    """+inf and the type's largest value act as 2**14, as documented; NaN does not hide."""
    q, k, v, _ = inputs(1, 2, 2, 200, 200, 64)
    top = table(32, 2)
    top[3] = 2.0 ** 14
    for x in (math.inf, torch.finfo(torch.bfloat16).max):
        other = top.clone()
        other[3] = x
        assert torch.equal(relative_attention(q[:, :, :n], k, v, other), relative_attention(q[:, :, :n], k, v, top))
    other[3] = math.nan
    o = relative_attention(q[:, :, :n], k, v, other)  # distance 3 behind: rows from 3 on see it
    assert torch.isnan(o[:, :, 3:]).all() and not torch.isnan(o[:, :, :3]).any()


def test_bias_gradient_against_differences():
    """The kernel's gradient of the table along a direction against central differences of the
    64-bit forward: their error is of the order of h**2, the bound is the gradient's own."""
    q, k, v, do = inputs(2, 3, 3, 200, 200, 64, size=0.125)
    bias = table(32, 3, size=1.0)
    leaf = bias.clone().requires_grad_(True)
    o = relative_attention(q, k, v, leaf, scale=1.0)
    (g,) = torch.autograd.grad(o, [leaf], do)
    bound = attend(q, k, v, do, bias=bias, both=True, scale=1.0)["dbias"][1]
    u = torch.randn(32, 3, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(2))
    at = lambda x: (attend(q, k, v, bias=x, both=True, scale=1.0)["o"][0] * do.double()).sum()  # noqa: E731
    h = 1e-5
    slope = (at(bias.double() + h * u) - at(bias.double() - h * u)) / (2 * h)
    assert abs((g.double() * u).sum() - slope) <= (bound * u.abs()).sum() + 1e-4


# ---- values that are not finite -------------------------------------------------------------

@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("B, H, Sq, Sk, D", [
    (1, 2, 1, 40, 64), (2, 2, 2, 5000, 128), (2, 16, 3, 20001, 128), (40, 16, 1, 700, 64),  # cluster, shares
    (2, 2, 130, 300, 64), (2, 2, 130, 300, 128), (1, 2, 130, 9000, 64), (1, 2, 260, 5000, 128),  # whole, split keys
])
def test_values_that_are_not_finite_are_seen(B, H, Sq, Sk, D, biased):
    """A visible query, key or value that is not finite makes the rows that see it NaN, and
    changes no other row."""
    q, k, v, _ = inputs(B, H, H, Sq, Sk, D)
    call = lambda q, k, v: relative_attention(q, k, v, table(32, H)) if biased else cross_attention(q, k, v)  # noqa: E731
    clean = call(q, k, v)

    def hit(o, rows):
        assert torch.isnan(o[0, 0, rows]).all()
        o = o.clone()
        o[0, 0, rows] = clean[0, 0, rows]
        assert torch.equal(o, clean)

    for x in (math.nan, math.inf):
        q2 = q.clone()
        q2[0, 0, Sq - 1, 3] = x
        hit(call(q2, k, v), slice(Sq - 1, Sq))
    for key in [*range(18), Sk // 2, Sk - 1]:  # all places in a group of columns
        k2 = k.clone()
        k2[0, 0, key, 5] = math.nan
        hit(call(q, k2, v), slice(None))
    k2 = k.clone()
    k2[0, 0, 17] = q[0, 0, 0].float().sign().to(torch.bfloat16) * math.inf  # a score of +inf in row 0
    assert torch.isnan(call(q, k2, v)[0, 0, 0]).all()
    v2 = v.clone()
    v2[0, 0, Sk - 1] = math.nan
    hit(call(q, k, v2), slice(None))


# ---- gradients that are wanted, determinism, graphs ---------------------------------------

@pytest.mark.parametrize("wanted", ["q", "k", "v", "b", "qk", "kb", "qb"])
def test_only_wanted_gradients(wanted):
    q, k, v, do = inputs(2, 4, 2, 150, 170, 64)
    bias = table(32, 4)
    want = attend(q, k, v, do, bias=bias, both=True, exact="b" in wanted)
    leaves = {n: t.clone().requires_grad_(n in wanted) for n, t in (("q", q), ("k", k), ("v", v), ("b", bias))}
    o = relative_attention(leaves["q"], leaves["k"], leaves["v"], leaves["b"], enable_gqa=True)
    o.backward(do)
    for n, name in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("b", "dbias")):
        if n in wanted:
            near(leaves[n].grad, want[name], name)
        else:
            assert leaves[n].grad is None


def test_no_grad_modes():
    q, k, v, _ = inputs(1, 2, 2, 100, 120, 64)
    want = cross_attention(q, k, v)
    q2 = q.clone().requires_grad_(True)
    with torch.no_grad():
        o = cross_attention(q2, k, v)
        assert not o.requires_grad and torch.equal(o, want)
    with torch.inference_mode():
        assert torch.equal(cross_attention(q2, k, v), want)
        assert torch.equal(torch.ops.ffa_b200.general_attention(q, k, v, None, None, None, 0, [], False, False, None), want)


def test_second_derivatives_are_refused():
    q, k, v, do = inputs(1, 2, 2, 100, 120, 64)
    q2 = q.clone().requires_grad_(True)
    o = cross_attention(q2, k, v)
    (g,) = torch.autograd.grad(o, [q2], do, create_graph=True)
    near(g, attend(q, k, v, do)["dq"], "dq")
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()


FORWARD_MODE = "forward-mode|forward AD"


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("Sq", [2, 100])
def test_forward_mode_derivatives_are_refused(Sq, grad):
    """Dual tensors, torch.func.jvp, a tangent of the output's gradient, and the registered operators."""
    q, k, v, do = inputs(1, 2, 2, Sq, 120, 64)
    bias = table(32, 2)
    general = _lib.ops().general
    calls = {
        "cross": lambda q, k, v, b: cross_attention(q, k, v),
        "relative": relative_attention,
        "general": lambda q, k, v, b: general(q, k, v, b, None, None, 0, list(bucket_borders(16, 128)), True, False, None),
        "lse": lambda q, k, v, b: _lib.ops().general_lse(q, k, v, None, None, None, 0, [], False, False, None,
                                                                 False)[0],
    }
    if grad:
        q.requires_grad_(True)
    for name, call in calls.items():
        for at in range(4 if name in ("relative", "general") else 3):
            args = [q, k, v, bias]
            def one(x):
                return call(*args[:at], x, *args[at + 1:])
            with pytest.raises((UnsupportedConfig, RuntimeError), match=FORWARD_MODE):
                torch.func.jvp(one, (args[at].detach(),), (torch.ones_like(args[at]),))
            with forward_ad.dual_level(), pytest.raises((UnsupportedConfig, RuntimeError), match=FORWARD_MODE):
                one(forward_ad.make_dual(args[at], torch.ones_like(args[at])))
    q2 = q.detach().clone().requires_grad_(True)
    o = cross_attention(q2, k, v)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(o, [q2], forward_ad.make_dual(do, torch.ones_like(do)), retain_graph=True)
        near(cross_attention(q, k, v), attend(q, k, v)["o"], "o")  # a level without tangents is no matter
        dual = forward_ad.make_dual(do, torch.ones_like(do))
        with forward_ad._set_fwd_grad_enabled(False):  # nor are tangents that nobody wants
            torch.autograd.grad(o, [q2], dual, retain_graph=True)
    near(torch.autograd.grad(o, [q2], do)[0], attend(q, k, v, do)["dq"], "dq")


@pytest.mark.parametrize("D", [64, 128])
def test_bitwise_deterministic(D):
    q, k, v, do = inputs(3, 4, 2, 700, 900, D, "bshd")
    bias = table(32, 4)
    lens = torch.tensor([900, 411, 77], dtype=torch.int32, device="cuda")
    def once():
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, bias)]
        o = relative_attention(*leaves, key_lengths=lens, enable_gqa=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, do), relative_attention(q[:, :, :2], k, v, bias, enable_gqa=True)]
    first = once()
    for _ in range(4):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    """Host threads on streams of their own get what they get one after another."""
    cases = [(inputs(2, 4, 2, 500, 3000, 64, seed=s), table(32, 4, seed=s)) for s in range(4)]
    lens = torch.tensor([3000, 1234], dtype=torch.int32, device="cuda")
    def work(case):
        (q, k, v, do), bias = case
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, bias)]
        o = relative_attention(*leaves, key_lengths=lens, enable_gqa=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, do),
                cross_attention(q[:, :, :1], k, v, key_lengths=lens, enable_gqa=True)]
    want = [work(c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * len(cases), []
    def run(n):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(3):
                    got[n] = work(cases[n])
            s.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)
    threads = [threading.Thread(target=run, args=(n,)) for n in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=120)
    assert not errors, errors
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_captured_steps_follow_their_lengths():
    """A decoding step captured once is replayed while the lengths grow, two graphs in turn."""
    q, k, v, _ = inputs(3, 4, 2, 1, 600, 64)
    bias = table(32, 4)
    graphs = []
    for n in range(2):
        lens = torch.tensor([10, 200, 400], dtype=torch.int32, device="cuda")
        offs = lens - 1
        step = lambda lens=lens, offs=offs: (  # noqa: E731
            relative_attention(q, k, v, bias, is_causal=True, query_offset=offs, key_lengths=lens, enable_gqa=True),
            cross_attention(q, k, v, key_lengths=lens, enable_gqa=True))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, lens, offs, out))
    for add in (0, 1, 150):
        for n, (g, lens, offs, out) in enumerate(graphs):
            lens += add + n
            offs.copy_(lens - 1)
            g.replay()
        torch.cuda.synchronize()
        for g, lens, offs, out in graphs:
            a = relative_attention(q, k, v, bias, is_causal=True, query_offset=lens - 1, key_lengths=lens, enable_gqa=True)
            b = cross_attention(q, k, v, key_lengths=lens, enable_gqa=True)
            assert torch.equal(out[0], a) and torch.equal(out[1], b)


@pytest.mark.parametrize("D", [64, 128])
def test_captured_training_step(D):
    q, k, v, do = inputs(2, 4, 2, 300, 420, D)
    bias = table(32, 4)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, bias)]
    def step():
        o = relative_attention(*leaves, enable_gqa=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for x in out:
        x.zero_()
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, out):
        assert torch.equal(a, b)


# ---- used together -----------------------------------------------------------------------

def test_encoder_decoder_layer():
    """An encoder layer over a padded batch, a decoder layer that attends to itself and to the
    encoder's states, trained as one; then the same tokens one by one over a cache."""
    torch.manual_seed(0)
    B, H, Se, Sd, D = 3, 4, 150, 90, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    enc = RelativeFlashAttention(H, scale=1.0, device="cuda")
    dec = RelativeFlashAttention(H, is_causal=True, scale=1.0, device="cuda")
    with torch.no_grad():
        for m in (enc, dec):
            m.bias.copy_(rnd(gen, 32, H))
    lens = torch.tensor([150, 60, 1], dtype=torch.int32, device="cuda")
    xe = rnd(gen, B, H, Se, D, size=0.3).requires_grad_(True)
    xd = rnd(gen, B, H, Sd, D, size=0.3).requires_grad_(True)
    states = enc(xe, xe, xe, key_lengths=lens)
    own = dec(xd, xd, xd)
    out = cross_attention(own, states, states, key_lengths=lens)
    do = rnd(gen, B, H, Sd, D)
    out.backward(do)
    # the same in 64 bits, from the kernels' own intermediate results (each operator is held
    # to its bound; the chain of gradients is that of autograd)
    near(states, attend(xe, xe, xe, bias=enc.bias, both=True, scale=1.0, lengths=lens)["o"], "states")
    near(own, attend(xd, xd, xd, bias=dec.bias, causal=True, scale=1.0)["o"], "own")
    w = attend(own, states, states, do, lengths=lens)
    near(out, w["o"], "out")
    d_states = (w["dk"][0].to(torch.bfloat16) + w["dv"][0].to(torch.bfloat16))
    e = attend(xe, xe, xe, d_states, bias=enc.bias, both=True, scale=1.0, lengths=lens)
    d = attend(xd, xd, xd, w["dq"][0].to(torch.bfloat16), bias=dec.bias, causal=True, scale=1.0)
    for got, parts, name in ((xe.grad, e, "xe"), (xd.grad, d, "xd")):
        want = parts["dq"][0] + parts["dk"][0] + parts["dv"][0]
        assert (got.double() - want).norm() <= 2e-2 * want.norm(), name  # four gates of 5e-3 in a row
    for got, parts, name in ((enc.bias.grad, e, "enc"), (dec.bias.grad, d, "dec")):
        assert (got.double() - parts["dbias"][0]).norm() <= 2e-2 * parts["dbias"][0].norm(), name
    # token by token over a cache, with lengths on the device
    with torch.no_grad():
        cache = torch.full((B, H, 128, D), math.nan, device="cuda", dtype=torch.bfloat16)
        n = torch.zeros(B, dtype=torch.int32, device="cuda")
        for t in range(Sd):
            cache[:, :, t] = xd[:, :, t]
            n += 1
            a = dec(xd[:, :, t:t + 1], cache, cache, query_offset=n - 1, key_lengths=n)
            near(a, tuple(x[:, :, t:t + 1] for x in attend_cached(d, xd, dec.bias)), "step", gate=1e-2)
            c = cross_attention(a, states, states, key_lengths=lens)
            near(c, attend(a, states, states, lengths=lens)["o"], "cross step", gate=1e-2)


def attend_cached(done, x, bias):
    """The full causal pass in 64 bits, once."""
    if "full" not in done:
        done["full"] = attend(x, x, x, bias=bias, causal=True, scale=1.0)["o"]
    return done["full"]
