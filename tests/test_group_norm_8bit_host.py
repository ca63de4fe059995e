"""Host side of group_norm_2d and the 8-bit operators: refusals, configurations, geometry.  CPU only."""

import dataclasses
import os
import re
import subprocess

import pytest
import torch

from spio_amd.build import CSRC_DIR, HIPCC_DEVICE_FLAGS, ROCM_HOME
from spio_amd.functional import activation_8bit, conv2d_gw8_8bit, group_norm_2d, pack_8bit, unpack_8bit
from spio_amd.functional.activation_8bit_function import Packed8bit, _is_dense
from spio_amd.functional.group_norm_2d_function import group_norm_2d_backward
from spio_amd.hip import DeviceAttributes
from spio_amd.kernels import (
    Activation8bitConfig,
    Activation8bitParams,
    GroupNorm2dParams,
    activation_8bit_kernel_factory,
    group_norm_2d_bwd_kernel_factory,
    group_norm_2d_kernel_factory,
)
from spio_amd.kernels.group_norm_2d_kernel import _span, is_legal
from spio_amd.layers import Activation8bit, GroupNorm2d
from tests.pointwise_reference import group_norm, pack_rows, values

ATTR = DeviceAttributes()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 16, 4, 4)
    with pytest.raises(ValueError):
        group_norm_2d(x, 4)
    with pytest.raises(ValueError):
        activation_8bit(x)
    with pytest.raises(ValueError):
        pack_8bit(x)
    with pytest.raises(ValueError):
        unpack_8bit(Packed8bit(torch.zeros(32, dtype=torch.int8), torch.zeros(1, dtype=torch.uint8), (32,), (1,), torch.float16))


@pytest.mark.parametrize("call", [
    lambda x: group_norm_2d(x, 5),
    lambda x: group_norm_2d(x, 0),
    lambda x: group_norm_2d(x, -4),
    lambda x: group_norm_2d(x[0], 4),
    lambda x: group_norm_2d(x[:, :4], 2),
    lambda x: group_norm_2d(x.double(), 4),
    lambda x: group_norm_2d(x, 4, eps=0.0),
    lambda x: group_norm_2d(x, 4, eps=float("inf")),
    lambda x: group_norm_2d(x, 4, eps=float("nan")),
    lambda x: group_norm_2d(x, 4, activation="tanh"),
    lambda x: group_norm_2d(x, 4, torch.ones(15)),
    lambda x: group_norm_2d(x, 4, None, torch.ones(16, 1)),
    lambda x: group_norm_2d(x, 4, torch.ones(16, dtype=torch.int32)),
    lambda x: activation_8bit(x, "none"),
    lambda x: activation_8bit(x.long()),
    lambda x: pack_8bit(x.double()),
    lambda x: unpack_8bit(Packed8bit(torch.zeros(31, dtype=torch.int8), torch.zeros(1, dtype=torch.uint8), (32,), (1,), x.dtype)),
    lambda x: unpack_8bit(Packed8bit(torch.zeros(32, dtype=torch.int8), torch.zeros(2, dtype=torch.uint8), (32,), (1,), x.dtype)),
    lambda x: unpack_8bit(Packed8bit(torch.zeros(32, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8), (32,), (1,), x.dtype)),
    lambda x: unpack_8bit(Packed8bit(torch.zeros(32, dtype=torch.int8), torch.zeros(1, dtype=torch.uint8), (4, 8), (16, 1), x.dtype)),
    lambda x: unpack_8bit(Packed8bit(torch.zeros(32, dtype=torch.int8), torch.zeros(1, dtype=torch.uint8), (32,), (1,), torch.int8)),
    lambda x: conv2d_gw8_8bit(x, torch.zeros(16, 8, 3, 3, requires_grad=True), groups=2),
    lambda x: group_norm_2d_backward(x, x, None, torch.zeros(2, 4, 3), 4, None, None, 1e-5, "none"),
])  # fmt: skip
def test_bad_arguments_are_refused(call):
    with pytest.raises((AssertionError, ValueError)):
        call(torch.zeros(2, 16, 4, 4))


def test_layers_refuse_activations_they_do_not_know():
    with pytest.raises(ValueError):
        GroupNorm2d(4, 16, activation="tanh")
    with pytest.raises(ValueError):
        Activation8bit("none")
    layer = GroupNorm2d(2, 8, activation="silu")
    x = torch.randn(2, 8, 3, 3)
    expected = torch.nn.functional.silu(torch.nn.functional.group_norm(x, 2))
    torch.testing.assert_close(layer(x), expected)
    assert torch.equal(Activation8bit("gelu")(x), torch.nn.functional.gelu(x))
    assert "silu" in repr(layer)


def test_dense_strides():
    assert _is_dense((2, 3, 4), (12, 4, 1)) and _is_dense((2, 3, 4), (1, 2, 6)) and _is_dense((1, 5), (99, 1))
    assert not _is_dense((2, 3), (6, 2)) and not _is_dense((2, 3), (0, 1)) and not _is_dense((2, 3), (2, 1))
    assert not _is_dense((4,), (-1,))


def _random_params(count):
    import random

    rng = random.Random(4)
    while count:
        c = 8 * rng.choice([1, 2, 3, 5, 9, 12, 24, 48, 96, 174, 512, rng.randint(1, 512)])
        groups = rng.choice([g for g in range(1, c + 1) if c % g == 0])
        yield GroupNorm2dParams(rng.choice([1, 2, 33]), c, rng.randint(1, 300), rng.randint(1, 300), groups, rng.randint(0, 2),
                                rng.randint(0, 3), 1e-5, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)  # fmt: skip
        count -= 1


def test_the_chosen_configurations_cover_every_shape():
    """Each is legal, holds the image or its stretches, gives workgroups within the limits of a launch, and needs
    no more LDS than a workgroup has."""
    for params in _random_params(400):
        for factory in (group_norm_2d_kernel_factory, group_norm_2d_bwd_kernel_factory):
            (config,) = factory.configs(params, ATTR)
            assert is_legal(params, config), (params, config)
            spec = factory.get_kernel_spec(params, config, ATTR)
            grid = spec.launch_params.grid[0]
            slices = -(-params.c // config.slice)
            stretches = -(-params.pixels // _span(params, config)) if config.split else 1
            assert grid == params.n * slices * stretches
            assert stretches * _span(params, config) >= params.pixels
            group = params.c // params.groups
            assert config.slice % group == 0 and (config.slice == params.c or config.slice % 32 == 0)
            # sums of two by channel, one row a lane row, where lanes do not fold; the groups' sums
            lanes = -(-config.slice // 8)
            lanes = -(-lanes // 4) * 4 if params.kept else lanes
            assert config.threads // lanes * lanes * 16 * 4 + 4 * config.slice * 4 <= 160 * 1024


def test_illegal_configurations_are_refused():
    params = GroupNorm2dParams(2, 64, 40, 40, 8)
    (config,) = group_norm_2d_kernel_factory.configs(params, ATTR)
    for change in ({"threads": 128}, {"units": 0}, {"slice": 24}, {"slice": 128}, {"units": 1, "split": 0, "slice": 64}):
        with pytest.raises(AssertionError):
            group_norm_2d_kernel_factory.get_kernel_spec(params, dataclasses.replace(config, **change), ATTR)
    for bad in ({"c": 60}, {"groups": 7}, {"c": 8192, "groups": 8}, {"eps": 0.0}, {"n": 0}):
        with pytest.raises(AssertionError):
            params_bad = dataclasses.replace(params, **bad)
            group_norm_2d_kernel_factory.get_kernel_spec(params_bad, config, ATTR)
    with pytest.raises(AssertionError):
        activation_8bit_kernel_factory.get_kernel_spec(Activation8bitParams(3), Activation8bitConfig(), ATTR)
    spec = activation_8bit_kernel_factory.get_kernel_spec(Activation8bitParams(), Activation8bitConfig(256, 4), ATTR)
    assert [spec.grid((n,))[0] for n in (1, 8192, 8193)] == [1, 1, 2]
    with pytest.raises(AssertionError):
        spec.grid((0,))
    with pytest.raises(AssertionError):
        spec.grid((1 << 38,))


def test_names_leave_out_the_images():
    """One file of compiled code serves all sizes of images."""
    a, b = GroupNorm2dParams(2, 64, 40, 40, 8), GroupNorm2dParams(7, 64, 12, 9, 8)
    assert a.encode() == b.encode()
    for field, value in (("c", 128), ("groups", 4), ("dtype", 1), ("activation", 2), ("eps", 1e-3), ("has_weight", False),
                         ("has_bias", False), ("kept", True)):  # fmt: skip
        other = dataclasses.replace(a, **{field: value}).encode()
        assert other != a.encode() and other.replace("_", "").isalnum()


def test_reference_formula_against_autograd():
    """The 64-bit reference of the GPU tests is the gradient of its own forward pass."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 12, 3, 2, generator=g, dtype=torch.float64)
    w, b = torch.randn(12, generator=g, dtype=torch.float64), torch.randn(12, generator=g, dtype=torch.float64)
    dy = torch.randn(2, 12, 3, 2, generator=g, dtype=torch.float64)
    for act in ("none", "relu", "silu", "gelu"):
        (_, dx, dw, db), *_ = group_norm(x, 3, w, b, 1e-5, act, dy)
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        z = torch.nn.functional.group_norm(leaves[0], 3, leaves[1], leaves[2])
        y = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act](z)
        for got, expected in zip((dx, dw, db), torch.autograd.grad(y, leaves, dy)):
            torch.testing.assert_close(got, expected, rtol=1e-10, atol=1e-10)


def test_the_8_bit_form_is_within_half_a_step():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(50, 77, generator=g) * torch.exp2(torch.randint(-30, 30, (50, 1), generator=g).float())
    codes, exponents = pack_rows(x)
    step = torch.exp2(exponents.double() - 133).repeat_interleave(32, -1)[:, :77]
    assert ((values(codes, exponents) - x.double()).abs() <= step / 2).all()
    assert exponents.shape == (50, 3) and codes.abs().max() <= 127


def test_a_record_for_other_images_is_passed_over(monkeypatch):
    """The kernels' names leave out the images: a configuration that is recorded under one is used only where it is
    the chosen one."""
    from spio_amd.kernels import tuner as tuner_object

    small, large = GroupNorm2dParams(1, 64, 8, 8, 8), GroupNorm2dParams(8, 64, 100, 100, 8)
    (wrong,), (right,) = (group_norm_2d_kernel_factory.configs(p, ATTR) for p in (large, small))
    assert wrong != right and is_legal(small, wrong)
    used = []
    monkeypatch.setattr("spio_amd.kernels.kernel_cache.compile_and_load_kernel",
                        lambda factory, params, config, *args, **kwargs: used.append(config))
    monkeypatch.setattr(tuner_object, "lookup", lambda attr, name: {"config": dataclasses.asdict(wrong)})
    monkeypatch.setenv("SPIO_TUNE", "1")
    tuner_object.best_kernel(group_norm_2d_kernel_factory, small, 0, ATTR)
    assert used == [right]


@pytest.mark.parametrize("factory", [group_norm_2d_kernel_factory, group_norm_2d_bwd_kernel_factory])
@pytest.mark.parametrize("params", [
    GroupNorm2dParams(5, 768, 14, 20, 32, 2, 2, has_bias=False, kept=True),
    GroupNorm2dParams(32, 48, 224, 224, 8, 0, 2),
    GroupNorm2dParams(1, 384, 50, 50, 3, 1, 3, kept=True),
])  # fmt: skip
def test_no_shift_of_64_bits_by_a_vector_register(factory, params, tmp_path):
    """The hardware takes a wrong number of places where that register is the last that a wave has: a conversion
    of a 64-bit integer, which has such a shift in it, made one of 240 values for some waves."""
    (config,) = factory.configs(params, ATTR)
    kernel = factory.make_kernel(params, config, ATTR)
    assert config.split
    out = str(tmp_path / "kernel.s")
    subprocess.run([os.path.join(ROCM_HOME, "bin", "hipcc"), "-S", "--cuda-device-only", *HIPCC_DEVICE_FLAGS, f"-I{CSRC_DIR}",
                    *[f"-D{k}={v}" for k, v in kernel.defines.items()], "-o", out,
                    os.path.join(CSRC_DIR, kernel.kernel_source_file)], check=True, capture_output=True)  # fmt: skip
    code = open(out).read()
    assert "buffer_load_dwordx" in code
    assert not re.findall(r"v_(?:lshl|lshr|ashr)rev_[bi]64\S* v\[\d+:\d+\], v\d+", code)
