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
    (lambda: _fwd(torch.zeros(1, dtype=torch.bfloat16).expand(1, 2 ** 31 - 2 ** 21, 1), groups=1), "too large"),
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


@pytest.mark.parametrize("which", ["each other, in part", "each other, bf16", "in x", "in dy", "gamma, in part", "beta, in part", "in stats"])
def test_gn_parameter_gradients_share_no_memory(which):
    c = 16
    x, dy, stats = torch.zeros(2, 3, c), torch.zeros(2, 3, c), torch.zeros(2, 4, 2)
    gamma, beta, dg, db, flat = torch.ones(c), torch.zeros(c), torch.zeros(c), torch.zeros(c), torch.zeros(3 * c)
    K._gn_check_writes(dg, db, x, dy, gamma, beta, stats)
    K._gn_check_writes(flat[:c], flat[c:2 * c], x, dy, flat[2 * c:], beta, stats)       # side by side
    if which == "each other, in part":
        dg, db = flat[:c], flat[c - 1:2 * c - 1]
    elif which == "each other, bf16":
        dg, db = flat.bfloat16()[:c], None
        db = dg[c - 1:]
    elif which == "in x":
        dg = x.view(-1)[c:2 * c]
    elif which == "in dy":
        db = dy.view(-1)[2 * c:3 * c]
    elif which == "gamma, in part":
        gamma, dg = flat[:c], flat[c // 2:c // 2 + c]
    elif which == "beta, in part":
        beta, dg = flat[4:4 + c], flat[:c]
    else:
        db = stats.view(-1)[:c]
    with pytest.raises(ValueError, match="share their memory"):
        K._gn_check_writes(dg, db, x, dy, gamma, beta, stats)


@pytest.mark.parametrize("bwd", [0, 1])
def test_rows_whose_count_would_pass_32_bits(bwd):
    """One channel and nearly 2^31 pixels: a piece's end, or a thread's next row behind it, is a negative number."""
    assert K._gn_workspace(1, 2 ** 31 - 2 ** 21 - 1, 1, 1, 0, bwd) > 0
    for hw in (2 ** 31 - 2 ** 21, 2 ** 31 - 2):
        with pytest.raises(ValueError, match="refuses"):
            K._gn_workspace(1, hw, 1, 1, 0, bwd)
