"""fast_attention and its operators know no forward-mode derivatives: they refuse dual tensors,
whose tangents they would otherwise drop without a word."""
import pytest
import torch
from torch.autograd import forward_ad

from fastflashattention_b200 import UnsupportedConfig, _lib, fast_attention, is_eligible
from fastflashattention_b200._kernel import fastflash_attn


class Cuda(torch.Tensor):
    """A CPU tensor that says it is on a CUDA device, so that the checks behind that one run."""
    is_cuda = True


@pytest.mark.parametrize("at", range(3))
def test_dual_tensors_are_refused(at):
    plain = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        args = [plain.clone().as_subclass(Cuda) for _ in range(3)]
        assert is_eligible(*args)
        args[at] = forward_ad.make_dual(plain, torch.ones_like(plain)).as_subclass(Cuda)
        assert not is_eligible(*args)
        with pytest.raises(UnsupportedConfig, match="forward-mode"):
            fast_attention(*args)


def test_registered_operators_refuse_tangents():
    """With a stand-in for the kernels: dual tensors and torch.func.jvp raise."""
    ops = _lib.ops()
    stand_in = torch.library.Library("ffa_b200", "IMPL")
    try:
        stand_in.impl("forward", lambda q, *_: q * 2, "CPU")
        stand_in.impl("forward_lse", lambda q, *_: (q * 2, q.sum(-1)), "CPU")
        q = torch.ones(1, 1, 2, 64)
        for call in (lambda x: ops.forward(x, q, q, False, None), lambda x: ops.forward_lse(q, q, x, False, None)[0]):
            with pytest.raises(NotImplementedError, match="forward AD"):
                torch.func.jvp(call, (q,), (q,))
            with forward_ad.dual_level():
                assert torch.equal(call(q), q * 2)
                with pytest.raises(NotImplementedError, match="forward AD"):
                    call(forward_ad.make_dual(q, q))
    finally:
        stand_in._destroy()


@pytest.mark.gpu
def test_on_the_gpu():
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, do = (torch.randn(1, 2, 128, 64, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(4))
    want = fast_attention(q, k, v)
    for call in (lambda x: fast_attention(q, x, v), lambda x: fastflash_attn(q, k, x, False),
                 lambda x: fastflash_attn(x, k, v, False, return_lse=True)[0]):
        with pytest.raises((UnsupportedConfig, RuntimeError), match="forward-mode|forward AD"):
            torch.func.jvp(call, (q,), (do,))
        with forward_ad.dual_level(), pytest.raises((UnsupportedConfig, RuntimeError), match="forward-mode|forward AD"):
            call(forward_ad.make_dual(q, do))
    leaf = q.clone().requires_grad_(True)
    o = fast_attention(leaf, k, v)
    (g,) = torch.autograd.grad(o, [leaf], do, retain_graph=True)
    with forward_ad.dual_level():
        assert torch.equal(fast_attention(q, k, v), want)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(o, [leaf], forward_ad.make_dual(do, do), retain_graph=True)
        dual = forward_ad.make_dual(do, do)
        with forward_ad._set_fwd_grad_enabled(False):  # tangents that nobody wants are no matter
            assert torch.equal(torch.autograd.grad(o, [leaf], dual, retain_graph=True)[0], g)
    assert torch.equal(torch.autograd.grad(o, [leaf], do)[0], g)
