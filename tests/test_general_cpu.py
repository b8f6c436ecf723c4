"""CPU: contracts of cross_attention and relative_attention, the bucket borders, and the
argument checks of the C ABI's general attention (they answer before touching the GPU)."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from fastflashattention_b200 import (RelativeFlashAttention, UnsupportedConfig, _lib, cross_attention,
                                     relative_attention)
from fastflashattention_b200._general import _bias_reason, _shape_reason, bucket_borders
from oracle.general_oracle import attend, bucket_of


class Cuda(torch.Tensor):
    """A CPU tensor that says it is on a CUDA device, so that the checks behind that one run."""
    is_cuda = True


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Cuda)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(UnsupportedConfig, match="CUDA"):
        cross_attention(q, q, q)
    with pytest.raises(UnsupportedConfig, match="CUDA"):
        relative_attention(q, q, q, torch.zeros(32, 2, dtype=torch.bfloat16))
    with pytest.raises(UnsupportedConfig, match="not a torch.Tensor"):
        cross_attention("q", q, q)


@pytest.mark.parametrize("q, k, v, extra, needle", [
    ((2, 4, 3, 64), (2, 4, 5, 64), (2, 4, 6, 64), {}, "key .* and value"),
    ((2, 4, 3, 64), (1, 4, 5, 64), (1, 4, 5, 64), {}, "same batch"),
    ((2, 4, 3, 64), (2, 4, 5, 32), (2, 4, 5, 32), {}, "same batch and head_dim"),
    ((2, 4, 3, 60), (2, 4, 5, 60), (2, 4, 5, 60), {}, "multiple of 8"),
    ((2, 4, 3, 136), (2, 4, 5, 136), (2, 4, 5, 136), {}, "multiple of 8"),
    ((2, 4, 3, 0), (2, 4, 5, 0), (2, 4, 5, 0), {}, "multiple of 8"),
    ((2, 4, 3, 64), (2, 2, 5, 64), (2, 2, 5, 64), {}, "enable_gqa"),
    ((2, 4, 3, 64), (2, 3, 5, 64), (2, 3, 5, 64), {"enable_gqa": True}, "multiple of key heads"),
    ((2, 4, 3, 64), (2, 0, 5, 64), (2, 0, 5, 64), {"enable_gqa": True}, "multiple of key heads"),
    ((2, 4, 3, 64), (2, 4, 5, 64), (2, 4, 5, 64), {"scale": math.inf}, "finite"),
    ((2, 4, 3, 64), (2, 4, 5, 64), (2, 4, 5, 64), {"scale": math.nan}, "finite"),
    ((4, 3, 64), (2, 4, 5, 64), (2, 4, 5, 64), {}, "dims"),
])
def test_shapes_outside_the_contract(q, k, v, extra, needle):
    with pytest.raises(UnsupportedConfig, match=needle):
        cross_attention(fake(*q), fake(*k), fake(*v), **extra)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_other_types_are_refused(dtype):
    q = fake(2, 4, 3, 64)
    with pytest.raises(UnsupportedConfig, match="bfloat16"):
        cross_attention(q, fake(2, 4, 5, 64, dtype=dtype), q)


@pytest.mark.parametrize("lengths, needle", [
    (torch.zeros(2, dtype=torch.int64), "int32"),
    (torch.zeros(3, dtype=torch.int32), "shape"),
    (torch.zeros(2, 1, dtype=torch.int32), "shape"),
    (torch.zeros(4, dtype=torch.int32)[::2], "contiguous"),
    ([3, 4], "not a torch.Tensor"),
])
def test_lengths_and_offsets_outside_the_contract(lengths, needle):
    q = fake(2, 4, 3, 64)
    assert _shape_reason(q, q, q, None, None, False) is None
    with pytest.raises(UnsupportedConfig, match=needle):
        cross_attention(q, q, q, key_lengths=lengths)
    if isinstance(lengths, torch.Tensor):
        with pytest.raises(UnsupportedConfig, match=needle):
            relative_attention(q, q, q, fake(32, 4), query_offset=lengths)


@pytest.mark.parametrize("bias, extra, needle", [
    (torch.zeros(32, 4), {}, "bfloat16"),
    (torch.zeros(32, 5, dtype=torch.bfloat16), {}, "column for each query head"),
    (torch.zeros(32, dtype=torch.bfloat16), {}, "column for each query head"),
    (torch.zeros(33, 4, dtype=torch.bfloat16), {}, "even"),
    (torch.zeros(2, 4, dtype=torch.bfloat16), {}, "buckets"),
    (torch.zeros(1, 4, dtype=torch.bfloat16), {"is_causal": True}, "buckets"),
    (torch.zeros(258, 4, dtype=torch.bfloat16), {}, "buckets"),
    (torch.zeros(32, 4, dtype=torch.bfloat16), {"max_distance": 8}, "max_distance"),
    (torch.zeros(32, 4, dtype=torch.bfloat16), {"max_distance": 1025}, "max_distance"),
    (torch.zeros(32, 4, dtype=torch.bfloat16), {"max_distance": 64.0}, "max_distance"),
    (torch.zeros(32, 4, dtype=torch.bfloat16), {"query_offset": 1.5}, "query_offset"),
    (torch.zeros(32, 4, dtype=torch.bfloat16), {"query_offset": 2 ** 29 + 1}, "2\\^29"),
    ("table", {}, "not a torch.Tensor"),
])
def test_bias_outside_the_contract(bias, extra, needle):
    q = fake(2, 4, 3, 64)
    with pytest.raises(UnsupportedConfig, match=needle):
        relative_attention(q, q, q, bias, **extra)


@pytest.mark.parametrize("dual", ["query", "key", "value", "bias"])
def test_forward_mode_derivatives_are_refused(dual):
    """The kernels know no tangents: a derivative of zero without a word would be wrong."""
    shapes = {"query": (1, 2, 3, 64), "key": (1, 2, 5, 64), "value": (1, 2, 5, 64), "bias": (32, 2)}
    with forward_ad.dual_level():
        t = {n: fake(*s) for n, s in shapes.items()}
        assert _shape_reason(t["query"], t["key"], t["value"], None, None, False) is None
        assert _bias_reason(t["query"], t["bias"], 128, None, False, 0) is None
        plain = torch.zeros(*shapes[dual], dtype=torch.bfloat16)
        t[dual] = forward_ad.make_dual(plain, torch.ones_like(plain)).as_subclass(Cuda)
        assert forward_ad.unpack_dual(t[dual]).tangent is not None
        with pytest.raises(UnsupportedConfig, match="forward-mode"):
            relative_attention(t["query"], t["key"], t["value"], t["bias"])
        if dual != "bias":
            with pytest.raises(UnsupportedConfig, match="forward-mode"):
                cross_attention(t["query"], t["key"], t["value"])


def test_registered_operators_refuse_tangents():
    """The operators themselves, with a stand-in for the kernel: dual tensors and torch.func.jvp
    raise, a level without tangents and a disabled forward mode do not, and backward raises."""
    ops = _lib.ops()
    stand_in = torch.library.Library("ffa_b200", "IMPL")
    try:
        stand_in.impl("general", lambda q, *_: q * 2, "CPU")
        q = torch.ones(1, 1, 2, 8)
        call = lambda q, bias=None: ops.general(q, q, q, bias, None, None, 0, [], False, False, None)  # noqa: E731
        with pytest.raises(NotImplementedError, match="forward AD"):
            torch.func.jvp(call, (q,), (q,))
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(q, q)
            for args in ((dual,), (q, dual)):
                with pytest.raises(NotImplementedError, match="forward AD"):
                    call(*args)
            assert torch.equal(call(q), q * 2)
            with forward_ad._set_fwd_grad_enabled(False):
                assert torch.equal(call(dual), q * 2)
        leaf = q.clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="not implemented"):
            call(leaf).sum().backward()
        with torch.no_grad():
            assert not call(leaf).requires_grad
    finally:
        stand_in._destroy()


def test_smallest_tables_are_inside_the_contract():
    q = fake(2, 4, 3, 64)
    assert _bias_reason(q, fake(4, 4), 2, None, False, 0) is None
    assert _bias_reason(q, fake(2, 4), 2, None, True, 0) is None
    assert _bias_reason(q, fake(256, 4), 1024, True, True, -5) is None


@pytest.mark.parametrize("side, distance", [(16, 128), (32, 128), (32, 256), (8, 64), (64, 800), (128, 1024), (2, 2),
                                            (3, 7), (5, 100)])
def test_borders_are_those_of_the_definition(side, distance):
    borders = bucket_borders(side, distance)
    assert len(borders) == side and borders[0] == 0 and list(borders) == sorted(borders) and borders[-1] <= distance
    r = torch.arange(distance + 50)
    by_border = torch.tensor([max(u for u in range(side) if borders[u] <= x) for x in r.tolist()])
    assert torch.equal(by_border, bucket_of(-r, side, distance, False))
    # the definition's logarithms in 64 bits, away from the borders that they hit exactly
    m = side // 2
    for x in r.tolist():
        if x >= m:
            y = m + (side - m) * math.log(x / m) / math.log(distance / m)
            if abs(y - round(y)) > 1e-9:
                assert by_border[x] == min(side - 1, math.floor(y)), x


def test_oracle_gradients_against_differences():
    """The oracle's gradients are those of its own forward: central differences of a weighted
    sum of the outputs along random directions (truncation is of the order of h**2)."""
    gen = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k, v, do, bias = rnd(2, 4, 5, 8), rnd(2, 2, 9, 8), rnd(2, 2, 9, 8), rnd(2, 4, 5, 8), rnd(8, 4)
    args = dict(max_distance=6, both=True, lengths=[7, 9], offsets=[1, -2])
    got = attend(q, k, v, do, bias=bias, **args)
    for name, x in (("dq", q), ("dk", k), ("dv", v), ("dbias", bias)):
        u, h = rnd(*x.shape), 1e-5
        def at(step):
            moved = {"dq": q, "dk": k, "dv": v, "dbias": bias, name: x + step * u}
            return (attend(moved["dq"], moved["dk"], moved["dv"], bias=moved["dbias"], **args)["o"][0] * do).sum()
        slope = (at(h) - at(-h)) / (2 * h)
        want = (got[name][0] * u).sum()
        assert abs(slope - want) < 1e-7 * (1 + abs(want)), name


def test_module_owns_its_table():
    m = RelativeFlashAttention(12, num_buckets=64, max_distance=256, is_causal=True, scale=1.0)
    assert m.bias.shape == (64, 12) and m.bias.dtype == torch.bfloat16 and m.bias.requires_grad
    assert [n for n, _ in m.named_parameters()] == ["bias"]
    assert "num_buckets=64" in repr(m) and "max_distance=256" in repr(m)


# ---- C ABI ---------------------------------------------------------------------------------

def problem(**changes):
    p = _lib.GenProblem(batch=2, q_heads=4, kv_heads=2, q_len=100, k_len=300, head_dim=64, causal=0, scale=0.125)
    borders = (ctypes.c_int * 16)(*bucket_borders(16, 128))
    p._borders = borders  # kept alive with the problem
    if changes.pop("with_bias", False):
        p.bias, p.buckets, p.both, p.borders = 16, 32, 1, borders
    for n, x in changes.items():
        setattr(p, n, x)
    return p


@pytest.mark.parametrize("changes, code, needle", [
    ({"head_dim": 36}, _lib.FFA_ERR_UNSUPPORTED, "head_dim"),
    ({"head_dim": 256}, _lib.FFA_ERR_UNSUPPORTED, "head_dim"),
    ({"batch": -1}, _lib.FFA_ERR_INVALID, "non-negative"),
    ({"q_heads": 5}, _lib.FFA_ERR_INVALID, "multiple of kv_heads"),
    ({"kv_heads": 0}, _lib.FFA_ERR_INVALID, "multiple of kv_heads"),
    ({"scale": math.inf}, _lib.FFA_ERR_INVALID, "finite"),
    ({"k_len": 1 << 29}, _lib.FFA_ERR_UNSUPPORTED, "2\\^29"),
    ({"query_offset": (1 << 29) + 1}, _lib.FFA_ERR_UNSUPPORTED, "query_offset"),
    ({"causal": 1}, _lib.FFA_ERR_UNSUPPORTED, "causal"),
    ({"with_bias": True, "buckets": 31}, _lib.FFA_ERR_UNSUPPORTED, "buckets"),
    ({"with_bias": True, "buckets": 300}, _lib.FFA_ERR_UNSUPPORTED, "buckets"),
    ({"batch": 1 << 20, "q_heads": 4096, "kv_heads": 4096}, _lib.FFA_ERR_UNSUPPORTED, "grid"),
])
def test_c_abi_refuses_problems(changes, code, needle):
    lib = _lib.load()
    p = problem(**changes)
    assert lib.ffa_gen_fwd_workspace(ctypes.byref(p), 0) == -1
    assert lib.ffa_gen_bwd_workspace(ctypes.byref(p)) == -1
    t = _lib.GenTensor(16, 64, 64, 64)
    r = ctypes.byref(t)
    rc = lib.ffa_gen_fwd(ctypes.byref(p), r, r, r, r, None, None, None, 0, None)
    import re
    assert rc == code and re.search(needle, _lib.last_error()), _lib.last_error()


def test_c_abi_refuses_borders_out_of_order():
    lib = _lib.load()
    for bad in ([1] + list(range(1, 16)), [0, 2, 1] + list(range(3, 16)), list(range(15)) + [1025]):
        p = problem(with_bias=True)
        p._borders = (ctypes.c_int * 16)(*bad)
        p.borders = p._borders
        assert lib.ffa_gen_fwd_workspace(ctypes.byref(p), 0) == -1
        assert "border" in _lib.last_error()


@pytest.mark.parametrize("tensor, needle", [
    ((0, 64, 64, 64), "null"), ((8, 64, 64, 64), "aligned"), ((16, 64, 64, 60), "strides"), ((16, 64, 0, 64), "strides"),
    ((16, -64, 64, 64), "strides"), ((16, 1 << 40, 64, 64), "strides"),
])
def test_c_abi_refuses_tensors(tensor, needle):
    lib = _lib.load()
    good, bad, p = _lib.GenTensor(16, 64, 64, 64), _lib.GenTensor(*tensor), problem()
    g, b = ctypes.byref(good), ctypes.byref(bad)
    for at in range(4):
        args = [g] * 4
        args[at] = b
        assert lib.ffa_gen_fwd(ctypes.byref(p), *args, None, None, None, 0, None) == _lib.FFA_ERR_INVALID
        assert needle in _lib.last_error()


def test_c_abi_wants_its_workspace():
    lib = _lib.load()
    p = problem(batch=1, q_heads=1, kv_heads=1, q_len=1, k_len=100000)
    need = lib.ffa_gen_fwd_workspace(ctypes.byref(p), 0)
    assert need > 0
    t = ctypes.byref(_lib.GenTensor(16, 64, 64, 64))
    for ws, size in ((None, need), (16, need - 1), (8, need)):
        assert lib.ffa_gen_fwd(ctypes.byref(p), t, t, t, t, None, None, ws, size, None) == _lib.FFA_ERR_INVALID
        assert "workspace" in _lib.last_error()
    assert lib.ffa_gen_bwd_workspace(ctypes.byref(problem())) > 0


def test_c_abi_backward_refusals():
    lib = _lib.load()
    p, t = problem(), ctypes.byref(_lib.GenTensor(16, 64, 64, 64))
    base = [ctypes.byref(p), t, t, t, t, None, t, 16]
    assert lib.ffa_gen_bwd(*base, t, t, None, None, 16, 1 << 40, None) == _lib.FFA_ERR_INVALID
    assert "together" in _lib.last_error()
    assert lib.ffa_gen_bwd(*base, t, t, t, 16, 16, 1 << 40, None) == _lib.FFA_ERR_INVALID
    assert "dbias" in _lib.last_error()
    base[7] = None
    assert lib.ffa_gen_bwd(*base, t, t, t, None, 16, 1 << 40, None) == _lib.FFA_ERR_INVALID


def test_c_abi_remainder_of_o_comes_with_a_bias():
    lib = _lib.load()
    t = ctypes.byref(_lib.GenTensor(16, 64, 64, 64))
    assert lib.ffa_gen_fwd(ctypes.byref(problem()), t, t, t, t, t, None, 16, 1 << 40, None) == _lib.FFA_ERR_INVALID
    assert "o_lo" in _lib.last_error()


def test_c_abi_nothing_to_do():
    lib = _lib.load()
    t = ctypes.byref(_lib.GenTensor(16, 64, 64, 64))
    for changes in ({"batch": 0}, {"q_heads": 0}, {"q_len": 0}):
        p = problem(**changes)
        assert lib.ffa_gen_fwd(ctypes.byref(p), t, t, t, t, None, None, None, 0, None) == _lib.FFA_OK


@pytest.mark.parametrize("causal", [0, 1])
def test_c_abi_no_query_heads_over_key_heads(causal):
    """A table of no heads has no data: a null bias is then no refusal."""
    lib = _lib.load()
    t = ctypes.byref(_lib.GenTensor(16, 64, 64, 64))
    p = problem(q_heads=0, causal=causal)
    assert lib.ffa_gen_fwd(ctypes.byref(p), t, t, t, t, None, None, None, 0, None) == _lib.FFA_OK
    assert lib.ffa_gen_bwd_workspace(ctypes.byref(p)) >= 0


def test_operators_are_registered():
    ops = _lib.ops()
    for name in ("general", "general_lse", "general_backward", "general_attention"):
        assert hasattr(ops, name), name
