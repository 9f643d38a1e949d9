"""The transformer-block operators (vectra_b200.block) beside the ordinary:
values that are not finite or far out, and uses that a call has to refuse.

Tolerances are those of test_block.py unless a test derives its own.
"""

import pytest
import torch

from tests.test_block import DEVICES
from tests.test_block import Rand
from vectra_b200 import block


# ---------------------------------------------------------------------------
# Forward mode
# ---------------------------------------------------------------------------
def _calls(device):
    """Each entry point with the tensors that can carry a tangent."""
    rand = Rand(3, device, torch.float32)
    cos, sin = block.rotation_tables(5, 8, device=device)
    return {
        'linear': (block.linear, [rand(3, 8), rand(4, 8), rand(4),
                                  rand(3, 4)]),
        'gated': (block.gated_linear, [rand(3, 8), rand(4, 8), rand(4, 8),
                                       rand(4), rand(4)]),
        'qk': (block.qk_norm_rope, [rand(2, 3, 5, 8), rand(2, 1, 5, 8), cos,
                                    sin, rand(8), rand(8)]),
    }


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('op', ['linear', 'gated', 'qk'])
@pytest.mark.parametrize('grad', [False, True])
def test_forward_mode_is_refused(device, op, grad):
    """A tangent in any argument raises (dropped, it would read as zero)."""
    fun, args = _calls(device)[op]
    ad = torch.autograd.forward_ad
    for i, t in enumerate(args):
        with ad.dual_level():
            tensors = [a.clone().requires_grad_(grad) for a in args]
            tensors[i] = ad.make_dual(tensors[i], torch.ones_like(t))
            with pytest.raises(NotImplementedError):
                fun(*tensors)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                fun(*tensors)
        if i == 0 and not grad:
            one = lambda a: fun(a, *args[1:])  # noqa: E731
            with pytest.raises(NotImplementedError):
                torch.func.jvp(one, (t,), (torch.ones_like(t),))
            with pytest.raises(NotImplementedError):
                torch.func.jacfwd(one)(t)
        # Outside the level the same tensors run.
        fun(*args)
