"""Forward-mode derivatives of the group norm and the 8-bit operators are refused: without a formula a tangent would come
out as zero or not at all."""

import pytest
import torch
from torch.autograd import forward_ad

from spio_amd import native
from spio_amd.functional import activation_8bit, conv2d_gw8_8bit, group_norm_2d

pytestmark = pytest.mark.gpu


def _tensors(requires_grad=False):
    x = torch.randn(2, 16, 6, 5, device="cuda").half().contiguous(memory_format=torch.channels_last)
    w = torch.randn(16, 8, 3, 3, device="cuda").half().contiguous(memory_format=torch.channels_last)
    return x, w.requires_grad_(requires_grad), torch.ones(16, device="cuda")


CALLS = {
    "norm": lambda x, w, b: group_norm_2d(x, 2, b, None, activation="silu"),
    "norm kept": lambda x, w, b: group_norm_2d(x, 2, b, b, checkpoint_8bit=True),
    "act": lambda x, w, b: activation_8bit(x),
    "conv": lambda x, w, b: conv2d_gw8_8bit(x, w, b, padding_y=1, padding_x=1, groups=2),
}


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("name", list(CALLS))
def test_forward_mode_is_refused(name, recorded, python):
    held = native.Bypass() if python else None
    x, w, b = _tensors(recorded)
    call = CALLS[name]
    expected = call(x, w, b).detach()
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(x.clone().requires_grad_(recorded), torch.randn_like(x)), w, b)
        if name != "act":
            with pytest.raises(NotImplementedError):
                call(x, w, forward_ad.make_dual(b, torch.randn_like(b)))
        assert torch.equal(call(x, w, b).detach(), expected)  # tensors without a tangent are as everywhere
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda t: call(t, w, b), (x,), (torch.randn_like(x),))
    if held:
        held.release()
