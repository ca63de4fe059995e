"""The native call path (csrc/spio_torch.cpp) of group_norm_2d, activation_8bit, pack_8bit, unpack_8bit and conv2d_gw8_8bit
against the Python definitions of the same operators, which run while a Bypass is held: equal results, the same
refusals, and gradients that notice what happened between the passes."""

import itertools
import threading

import pytest
import torch

from spio_amd import native
from spio_amd.functional import activation_8bit, conv2d_gw8_8bit, group_norm_2d, pack_8bit, unpack_8bit
from spio_amd.kernels import KernelParamsLogger
from spio_amd.kernels.kernel import LaunchTimer

pytestmark = pytest.mark.gpu
CL = torch.channels_last
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _norm(dtype=torch.float16, kept=False, vectors="wb", grads="xwb", c=24, hw=(9, 7), vector_dtype=torch.float32):
    torch.manual_seed(3)
    x = torch.randn(3, c, *hw, device="cuda").to(dtype).contiguous(memory_format=CL).requires_grad_("x" in grads)
    v = {k: torch.rand(c, device="cuda").to(vector_dtype).requires_grad_(k in grads) if k in vectors else None for k in "wb"}
    return [x, v["w"], v["b"]], lambda x, w, b: group_norm_2d(x, 4, w, b, 1e-5, "silu", kept)


def _act(dtype=torch.float16):
    torch.manual_seed(4)
    x = torch.randn(5, 33, 7, device="cuda").to(dtype).requires_grad_()
    return [x], lambda x: activation_8bit(x, "gelu")


def _conv(autocast=False):
    torch.manual_seed(5)
    dtype = torch.float32 if autocast else torch.float16
    x = torch.randn(3, 24, 9, 7, device="cuda").to(dtype).contiguous(memory_format=CL).requires_grad_()
    w = (torch.randn(24, 8, 3, 3, device="cuda") * 0.1).to(dtype).contiguous(memory_format=CL).requires_grad_()
    b = torch.randn(24, device="cuda").requires_grad_()

    def call(x, w, b):
        with torch.autocast("cuda", dtype=torch.float16, enabled=autocast):
            return conv2d_gw8_8bit(x, w, b, padding_y=1, padding_x=1, groups=3)

    return [x, w, b], call


CALLS = {
    "norm": _norm, "norm kept": lambda: _norm(kept=True), "norm large": lambda: _norm(hw=(60, 57), c=64),
    "norm float32": lambda: _norm(torch.float32, True), "act": _act, "act bf16": lambda: _act(torch.bfloat16),
    "conv": _conv, "conv autocast": lambda: _conv(True),
}  # fmt: skip


def _run(leaves, call, dy=None):
    y = call(*leaves)
    wanted = [t for t in leaves if t is not None and t.requires_grad]
    if dy is None:
        dy = torch.randn(y.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(y.dtype)
    return [y.detach(), *torch.autograd.grad(y, wanted, dy)]


def _same(got, expected, exact=True):
    assert len(got) == len(expected)
    for a, e in zip(got, expected):
        assert a.dtype == e.dtype and a.shape == e.shape and a.stride() == e.stride()
        if exact:
            assert torch.equal(a, e)
        else:  # weight gradients of a convolution: atomic sums, and a rounding on the way in the Python operator
            torch.testing.assert_close(a.float(), e.float(), rtol=4e-3, atol=2e-3 * float(e.float().abs().max()))


@pytest.mark.parametrize("name", list(CALLS))
def test_native_and_python_agree(name):
    leaves, call = CALLS[name]()
    got = _run(leaves, call)
    held = native.Bypass()
    expected = _run(leaves, call)
    held.release()
    _same(got, expected, exact="conv" not in name)
    with torch.no_grad():
        assert torch.equal(call(*leaves), got[0]) or name == "norm float32"  # (padded lanes: another order of sums)


@pytest.mark.parametrize("vectors", ["", "w", "b", "wb"])
@pytest.mark.parametrize("kept", [False, True])
def test_every_choice_of_gradients(vectors, kept):
    """Whatever of the input, weight and bias is there and wants a gradient gets its own."""
    full_leaves, call = _norm(kept=kept, vectors=vectors, grads="x" + vectors)
    full = dict(zip("yx" + vectors, _run(full_leaves, call)))
    for r in range(1, 2 + len(vectors)):
        for grads in itertools.combinations("x" + vectors, r):
            leaves, call = _norm(kept=kept, vectors=vectors, grads="".join(grads))
            for key, g in zip(("y", *grads), _run(leaves, call)):
                assert torch.equal(g, full[key]), (grads, key)


@pytest.mark.parametrize("vector_dtype", [torch.float16, torch.bfloat16])
def test_vectors_of_other_types(vector_dtype):
    leaves, call = _norm(vector_dtype=vector_dtype)
    got = _run(leaves, call)
    assert got[2].dtype == got[3].dtype == vector_dtype
    held = native.Bypass()
    _same(got, _run(leaves, call))
    held.release()


_HOOKS = {
    "relaid": lambda: torch.autograd.graph.saved_tensors_hooks(
        lambda t: t.detach().clone(memory_format=torch.contiguous_format), lambda t: t),
    "host": lambda: torch.autograd.graph.save_on_cpu(),
    "transposed": lambda: torch.autograd.graph.saved_tensors_hooks(
        lambda t: t.detach().transpose(0, -1).contiguous(), lambda t: t.transpose(0, -1)),
}  # fmt: skip


@pytest.mark.parametrize("hooks", list(_HOOKS))
@pytest.mark.parametrize("name", ["norm", "norm kept", "act", "conv"])
def test_saved_tensors_may_come_back_in_another_layout(name, hooks):
    leaves, call = CALLS[name]()
    expected = _run(leaves, call)
    dy = torch.randn(expected[0].shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(expected[0].dtype)
    with _HOOKS[hooks]():
        y = call(*leaves)
    got = [y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], dy)]
    _same(got, expected, exact=name != "conv")


@pytest.mark.parametrize("bypass", [False, True])
@pytest.mark.parametrize("name", ["norm", "norm kept", "act", "conv"])
def test_second_derivatives_are_refused(name, bypass):
    """Where the backward pass has what it would take (the input itself) when they are asked for, else before."""
    leaves, call = CALLS[name]()
    held = native.Bypass() if bypass else None
    try:
        y = call(*leaves)
        with pytest.raises(RuntimeError):
            grads = torch.autograd.grad(y, leaves, torch.ones_like(y), create_graph=True)
            torch.autograd.grad(grads[0].float().sum(), leaves)
    finally:
        if held:
            held.release()


def test_a_changed_input_is_noticed():
    leaves, call = _norm()
    x = leaves[0] * 1
    y = call(x, *leaves[1:])
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    leaves, call = _norm(kept=True)  # the checkpoint is a copy; the vectors are not
    x, w = leaves[0] * 1, leaves[1] * 1
    expected = torch.autograd.grad(call(x, w, leaves[2]), leaves[0], torch.ones_like(x))
    x = leaves[0] * 1
    y = call(x, w, leaves[2])
    x.add_(1)
    assert torch.equal(torch.autograd.grad(y, leaves[0], torch.ones_like(x))[0], expected[0])
    y = call(leaves[0], w, leaves[2])
    w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_retained_graphs_and_repeated_tensors():
    leaves, call = _norm(kept=True)
    y = call(*leaves)
    dy = torch.randn_like(y)
    once, twice = (torch.autograd.grad(y, leaves, dy, retain_graph=True) for _ in range(2))
    _same(twice, once)
    x, w, _ = leaves
    y = group_norm_2d(x, 4, w, w)  # one tensor in two places: the sum of both gradients
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    parts = torch.autograd.grad(group_norm_2d(x, 4, w, leaves[1].detach().clone().requires_grad_()), [w], dy)
    bias_part = dy.float().sum((0, 2, 3))
    torch.testing.assert_close(dw, parts[0] + bias_part, rtol=1e-4, atol=1e-4)


def test_calls_from_several_threads():
    """Each on a stream of its own: workspaces and plans are not shared between calls that overlap."""
    leaves, call = _norm(hw=(60, 57), c=64, kept=True)
    dy = torch.randn(3, 64, 60, 57, device="cuda").half().contiguous(memory_format=CL)
    expected = _run(leaves, call, dy)
    torch.cuda.synchronize()
    results = {}

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            mine = [t.detach().clone().requires_grad_() for t in leaves]
            for _ in range(10):
                results[i] = _run(mine, call, dy)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        _same(results[i], expected)


def test_a_backward_pass_on_another_stream():
    """The engine runs a node on the stream of its forward pass, whatever the current one is then."""
    leaves, call = _norm(kept=True)
    expected = _run(leaves, call)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = call(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    dy = torch.randn(y.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(y.dtype)
    got = torch.autograd.grad(y, leaves, dy)
    torch.cuda.synchronize()
    _same(got, expected[1:])


@pytest.mark.parametrize("recorder", [KernelParamsLogger, LaunchTimer])
@pytest.mark.parametrize("name", ["norm kept", "norm large", "act", "conv"])
def test_recorders_see_the_launches(name, recorder):
    leaves, call = CALLS[name]()
    expected = _run(leaves, call)
    with recorder() as seen:
        got = _run(leaves, call)
    _same(got, expected, exact=name != "conv")
    found = seen.get_logged_params() if recorder is KernelParamsLogger else seen.averages()
    assert len(found) >= 2


def _profiled(name):
    leaves, call = CALLS[name]()
    _run(leaves, call)
    with torch.autograd.profiler.profile(record_shapes=True, use_device=None) as profile:
        _run(leaves, call)
    return {e.name for e in profile.function_events if e.name.startswith("spio::")}


@pytest.mark.parametrize("name", ["norm", "norm kept", "act"])
def test_profiles_show_the_operators(name):
    seen = _profiled(name)
    held = native.Bypass()
    expected = _profiled(name)
    held.release()
    assert len(expected) == 2 and seen == expected


def test_pack_and_unpack():
    torch.manual_seed(7)
    for dtype in DTYPES:
        x = torch.randn(3, 24, 5, 7, device="cuda").to(dtype)
        for t in (x, x.contiguous(memory_format=CL), x.permute(2, 0, 3, 1), x.reshape(-1)[3:90]):
            packed = pack_8bit(t)
            back = unpack_8bit(packed)
            held = native.Bypass()
            again = pack_8bit(t)
            assert torch.equal(packed.codes, again.codes) and torch.equal(packed.exponents, again.exponents)
            assert packed[2:] == again[2:]
            expected = unpack_8bit(again)
            held.release()
            assert back.stride() == expected.stride() and torch.equal(back, expected)
            # strides that leave a gap or overlap, sizes that do not fit: refused on both paths
            for bad in (packed._replace(strides=tuple(2 * s for s in packed.strides)),
                        packed._replace(shape=(*packed.shape, 2), strides=(*packed.strides, 1)),
                        packed._replace(codes=packed.codes[1:]), packed._replace(exponents=packed.exponents[1:]),
                        packed._replace(dtype=torch.float64)):  # fmt: skip
                with pytest.raises((AssertionError, ValueError)):
                    unpack_8bit(bad)


def test_vectors_off_16_bytes():
    """float32 vectors are read where they are: four bytes behind a border too."""
    leaves, call = _norm()
    expected = _run(leaves, call)
    off = [torch.cat([t.detach()[:1], t.detach()])[1:].requires_grad_() for t in leaves[1:]]
    assert all(t.data_ptr() % 16 == 4 for t in off)
    _same(_run([leaves[0], *off], call), expected)


def test_inference_mode():
    leaves, call = _norm(kept=True)
    expected = call(*leaves)
    with torch.inference_mode():
        x = leaves[0].detach().clone()
        assert torch.equal(call(x, *leaves[1:]), call(*leaves))
        torch.testing.assert_close(call(x, *leaves[1:]), expected, rtol=2e-3, atol=2e-3)
        y = activation_8bit(x, "silu")
        assert torch.equal(unpack_8bit(pack_8bit(x)), unpack_8bit(pack_8bit(leaves[0])))
    torch.testing.assert_close(y, torch.nn.functional.silu(leaves[0]), rtol=2e-3, atol=2e-3)


@pytest.mark.parametrize("hw", [(9, 7), (60, 57)])
def test_the_static_workspace_serves_both_passes(hw):
    """Launches of the kernels that must not allocate: whole images and stretches."""
    from spio_amd.kernels import GroupNorm2dParams, group_norm_2d_bwd_kernel_factory, group_norm_2d_kernel_factory

    leaves, call = _norm(c=64, hw=hw)
    dy = torch.randn(3, 64, *hw, device="cuda").half().contiguous(memory_format=CL)
    y, dx, dw, db = _run(leaves, call, dy)
    x, w, b = (t.detach() for t in leaves)
    params = GroupNorm2dParams(3, 64, *hw, 4, activation=2)
    out, grad, sums = torch.empty_like(x), torch.empty_like(x), torch.empty(2, 64, device="cuda")
    stats = torch.empty(3, 4, 2, device="cuda")
    forward = group_norm_2d_kernel_factory.get_kernel(params, x.device)
    forward.launch(out, None, None, stats, x, w, b, params.pixels, 3, static_workspace=True)
    backward = group_norm_2d_bwd_kernel_factory.get_kernel(params, x.device)
    backward.launch(sums, grad, x, None, dy, stats, w, b, params.pixels, 3, static_workspace=True)
    _same([out, grad, sums[0], sums[1]], [y, dx, dw, db])


def test_replays_of_a_captured_convolution():
    leaves, call = _conv()
    dy = torch.randn(3, 24, 9, 7, device="cuda").half().contiguous(memory_format=CL)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(leaves, call, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = _run(leaves, call, dy)
    for seed in range(3):
        torch.manual_seed(seed)
        with torch.no_grad():
            leaves[0].copy_(torch.randn(3, 24, 9, 7, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        _same(out, _run(leaves, call, dy), exact=False)


def test_a_compiled_convolution():
    leaves, call = _conv()
    compiled = torch.compile(lambda x, w, b: conv2d_gw8_8bit(x, w, b, padding_y=1, padding_x=1, groups=3), backend="aot_eager")
    _same(_run(leaves, compiled), _run(leaves, call), exact=False)


def test_arguments_by_name_and_what_the_native_path_leaves_to_python():
    leaves, call = _norm()
    x, w, b = leaves
    expected = group_norm_2d(x, 4, w, b, 1e-3, "gelu", True)
    assert torch.equal(group_norm_2d(inputs=x, num_groups=4, weight=w, bias=b, eps=1e-3, activation="gelu", checkpoint_8bit=True), expected)
    assert torch.equal(group_norm_2d(x, 4, w, b, eps=1e-3, activation="gelu", checkpoint_8bit=1), expected)
    with pytest.raises(AssertionError):
        group_norm_2d(x, 5, w, b)
    with pytest.raises(AssertionError):
        group_norm_2d(x, 4, w, b, activation="tanh")
    with pytest.raises(AssertionError):
        activation_8bit(x, "none")
    one = group_norm_2d(x, 4, w, b, 1)  # eps as an integer
    assert torch.equal(one, group_norm_2d(x, 4, w, b, 1.0))


def test_a_block_of_all_of_them_and_its_tuning(monkeypatch, tmp_path):
    """A convolution, a norm and an activation that keep their inputs in 8 bits, one behind the other: gradients within
    what the checkpoints' half steps change, and the same results after the model's kernels were timed and recorded."""
    from spio_amd.layers import Activation8bit, Conv2dGw8, GroupNorm2d
    from spio_amd.tune import tune_model

    monkeypatch.setenv("SPIO_TUNE_DB", str(tmp_path / "tuned.json"))
    torch.manual_seed(8)
    conv = Conv2dGw8(96, 96, 3, padding=1, groups=12, bias=False)
    norm = GroupNorm2d(12, 96, activation="silu")
    block = torch.nn.Sequential(conv, norm, torch.nn.Conv2d(96, 192, 1), Activation8bit("gelu"))
    block = block.cuda().half().to(memory_format=CL)
    x = torch.randn(4, 96, 20, 18, device="cuda").half().contiguous(memory_format=CL)

    def gradients(kept):
        conv.checkpoint_8bit = norm.checkpoint_8bit = kept
        block.zero_grad()
        y = block(x)
        y.float().square().mean().backward()
        return [y.detach().clone(), *(p.grad.clone() for p in block.parameters())]

    plain, kept = gradients(False), gradients(True)
    assert torch.equal(plain[0], kept[0])
    for a, b in zip(plain[1:], kept[1:]):
        # a checkpoint is off by 1/255 of a block's largest value (five deviations, say) at most, and an input by
        # 1/50 of its deviation so; as a vector a gradient is off by no more than these add up to in the two kept inputs
        assert (a - b).float().norm() <= 0.04 * a.float().norm()
    results = tune_model(block, [x], iters=1, warmup=1)
    names = {r["kernel"].split("__")[0] for r in results}
    assert {"spio_group_norm_2d", "spio_group_norm_2d_bwd", "spio_activation_8bit", "spio_activation_8bit_bwd", "spio_pack_8bit",
            "spio_unpack_8bit", "spio_conv2d_gw8_fprop"} <= names  # fmt: skip
    assert all(r["config"] is not None for r in results)
    for a, b in zip(kept, gradients(True)):
        torch.testing.assert_close(a, b, rtol=2e-2, atol=2e-2 * float(a.abs().max()))
