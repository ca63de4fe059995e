"""What the operators over sequences of tokens share: how their tensors lie in memory."""

from typing import Optional, Tuple

import torch

from ..kernels.group_norm_2d_kernel import DTYPES

MAX_ROW = 1 << 27  # bytes from row to row of a tensor that is read in tiles


def check_tokens(what: str, **tensors: Optional[torch.Tensor]):
    """Types and devices of the tensors of an operator: one of the three types, the first one's, on its device."""
    first = next(iter(tensors.values()))
    for name, t in tensors.items():
        assert t is None or t.dtype in DTYPES, f"{what} takes float16, bfloat16 or float32 tensors"
        assert t is None or t.dtype == first.dtype, f"{what}: {name} must have the type of the first tensor"
        assert t is None or t.device == first.device, f"{what}: {name} must be on the first tensor's device"


def check_parameters(what: str, like: torch.Tensor, **parameters):
    """Shapes of parameters, which may have another float type: name=(tensor, shape)."""
    for name, (t, shape) in parameters.items():
        assert t is None or (t.is_floating_point() and tuple(t.shape) == tuple(shape)), f"{what}: {name} must be {list(shape)}"
        assert t is None or t.device == like.device, f"{what}: {name} must be on the first tensor's device"


def require_gpu(what: str, t: torch.Tensor):
    if t.device.type != "cuda":
        raise ValueError(f"spio::{what} runs on the GPU only")


def rows_of(t: Optional[torch.Tensor], step: int = 1) -> Tuple[Optional[torch.Tensor], int]:
    """[sequences, tokens, values] (or [sequences, values]) as rows of values that are equally far apart: the tensor itself,
    or a copy without gaps where it is not that, where rows do not start on 16 bytes though `step` (8) values are loaded at
    once, or where a tile of eight rows that are read by their distance to the first would pass 31 bits.  Also their distance
    in values."""
    if t is None:
        return None, 0
    *lead, last = t.shape
    sizes = [(size, stride) for size, stride in zip(lead, t.stride()) if size != 1]
    row = sizes[-1][1] if sizes else last
    even = all(outer[1] == inner[0] * inner[1] for outer, inner in zip(sizes, sizes[1:]))
    size = row * t.element_size()
    fits = size < MAX_ROW if step == 1 else size % 16 == 0 and t.data_ptr() % 16 == 0
    if even and fits and (last == 1 or t.stride(-1) == 1):
        return t, row
    t = t.clone(memory_format=torch.contiguous_format)
    return t, last


def vector(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A parameter in float32 without gaps."""
    return None if t is None else t.detach().float().contiguous()


def refuse_state_gradients(*tensors):
    """A state passes from call to call without a history; a gradient of it would silently be missing."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("no gradients pass through a state: detach it")


def refuse_inference_state(t: torch.Tensor):
    """As torch's own operators do, which keep no versions of such tensors."""
    if t.is_inference() and not torch.is_inference_mode_enabled():
        raise RuntimeError("a state that was made in inference mode is updated there only")


def _extent(t: torch.Tensor) -> Tuple[int, int]:
    """Addresses of a tensor's first byte and behind its last one."""
    last = sum((size - 1) * stride for size, stride in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the bytes from a tensor's first to its last value meet another's."""
    if a.numel() == 0 or b.numel() == 0 or a.device != b.device:
        return False
    (a_first, a_end), (b_first, b_end) = _extent(a), _extent(b)
    return a_first < b_end and b_first < a_end


def check_out_state(what: str, state: torch.Tensor, out_state: torch.Tensor, *inputs):
    """Where the state of a step goes: a tensor like it, the same one or one that shares nothing with it; nor with the other
    inputs."""
    assert out_state.shape == state.shape and out_state.dtype == state.dtype and out_state.device == state.device, (
        f"{what}: out_state must be like state")  # fmt: skip
    assert state.is_contiguous() and out_state.is_contiguous(), f"{what}: states must have no gaps"
    assert state.data_ptr() == out_state.data_ptr() or not overlap(state, out_state), f"{what}: out_state overlaps state"
    for t in inputs:
        assert t is None or not overlap(t, out_state), f"{what}: out_state overlaps an input"
