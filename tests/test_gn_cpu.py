"""Group norm + activation on the CPU: what the entry points refuse, before anything touches a device."""
import pytest
import torch

from distributed_training_pytorch_amd.ops import kernels as K


def _fwd(x, groups=4, act="relu", gamma=None, beta=None):
    c = x.shape[-1] if x.dim() else 1
    return K.gn_fwd(x, torch.ones(c) if gamma is None else gamma, torch.zeros(c) if beta is None else beta, groups, act=act)


@pytest.mark.parametrize("call,what", [
    (lambda: _fwd(torch.zeros(2, 3, 16, dtype=torch.float64)), "bf16, f16 or f32"),
    (lambda: _fwd(torch.zeros(16)), r"\[N, \.\.\., C\]"),
    (lambda: _fwd(torch.zeros(2, 3, 16), act="tanh"), "act must be one of"),
    (lambda: _fwd(torch.zeros(2, 3, 16), groups=5), "multiple of groups"),
    (lambda: _fwd(torch.zeros(2, 3, 16), groups=0), "multiple of groups"),
    (lambda: _fwd(torch.zeros(1, 1, 4100)), "at most 4096"),
    (lambda: _fwd(torch.zeros(2, 0, 16)), "no values"),
    (lambda: _fwd(torch.zeros(1, dtype=torch.bfloat16).expand(1, 2 ** 27, 16)), "too large"),
    (lambda: _fwd(torch.zeros(2, 3, 16), gamma=torch.ones(15)), "gamma / beta"),
    (lambda: _fwd(torch.zeros(2, 3, 16), beta=torch.ones(16, dtype=torch.bfloat16)), "gamma / beta"),
    (lambda: _fwd(torch.zeros(2, 3, 16)), "must be a CUDA tensor"),
    (lambda: K.gn_bwd(torch.zeros(2, 3, 16), torch.zeros(2, 3, 8), torch.ones(16), torch.ones(16), None, 4, None, None),
     "dy must have"),
    (lambda: K.gn_bwd(torch.zeros(2, 3, 16), torch.zeros(2, 3, 16, dtype=torch.bfloat16), torch.ones(16), torch.ones(16),
                      None, 4, None, None), "dy must have"),
])
def test_gn_refusals(call, what):
    with pytest.raises(ValueError, match=what):
        call()


@pytest.mark.parametrize("bwd", [0, 1])
def test_more_threads_than_a_launch_holds(bwd):
    """2^24 one-pixel images and up: 256 threads each are 2^32 (4 million are fine: their groups fit one slab)."""
    assert K._gn_workspace(1 << 22, 1, 32, 4, 0, bwd) == bwd * (1 << 22) * 64
    with pytest.raises(ValueError, match="refuses"):
        K._gn_workspace(1 << 24, 1, 32, 4, 0, bwd)
    with pytest.raises(ValueError, match="refuses"):
        K._gn_workspace(1 << 22, 1, 4096, 4096, 0, bwd)
