"""Host side of the operators over sequences of tokens: refusals, geometry, structures of arguments, frequencies, compiled
code.  CPU only."""

import math
import os
import re
import subprocess

import pytest
import torch

from spio_amd import kernels, native
from spio_amd.build import CSRC_DIR, HIPCC_DEVICE_FLAGS, ROCM_HOME
from spio_amd.functional import (
    causal_conv1d,
    causal_conv1d_step,
    head_norm_rotary,
    rotary,
    rotary_frequencies,
    selective_scan,
    selective_scan_step,
)
from spio_amd.functional.causal_conv1d_function import causal_conv1d_forward
from spio_amd.functional.head_norm_rotary_function import _heads_of
from spio_amd.functional.selective_scan_function import selective_scan_forward
from spio_amd.functional.token_rows import overlap, rows_of
from spio_amd.hip import DeviceAttributes
from spio_amd.kernels.causal_conv1d_kernel import slice_tokens
from spio_amd.kernels.head_norm_rotary_kernel import grid_of, lanes_of, parts_of
from spio_amd.kernels.selective_scan_kernel import chunk_tokens, tile_tokens
from spio_amd.kernels.token_args import Arguments, fields_of
from spio_amd.layers import CausalConv1d, HeadNormRotary, SelectiveScan

X, W = torch.zeros(2, 5, 16), torch.ones(16, 4)
A, ROWS = -torch.ones(16, 3), torch.zeros(2, 5, 3)
Q, POSITIONS, FREQUENCIES = torch.zeros(2, 5, 4, 32), torch.arange(5), rotary_frequencies(32)


def test_cpu_tensors_are_refused():
    for call in (
        lambda: causal_conv1d(X, W),
        lambda: causal_conv1d_step(X[:, 0], torch.zeros(2, 3, 16), W),
        lambda: selective_scan(X, X, A, ROWS, ROWS),
        lambda: selective_scan_step(X[:, 0], torch.zeros(2, 16, 3), X[:, 0], A, ROWS[:, 0], ROWS[:, 0]),
        lambda: rotary(Q, Q, POSITIONS, FREQUENCIES),
        lambda: head_norm_rotary(Q, Q, torch.ones(32), torch.ones(32), POSITIONS, FREQUENCIES),
    ):
        with pytest.raises(ValueError, match="GPU only"):
            call()


@pytest.mark.parametrize("call", [
    lambda: causal_conv1d(X[0], W),
    lambda: causal_conv1d(X[..., :12], W[:12]),
    lambda: causal_conv1d(X, W[:, 0]),
    lambda: causal_conv1d(X, torch.ones(16, 1)),
    lambda: causal_conv1d(X, torch.ones(16, 9)),
    lambda: causal_conv1d(X, W.long()),
    lambda: causal_conv1d(X, W, torch.ones(15)),
    lambda: causal_conv1d(X, W, None, "relu"),
    lambda: causal_conv1d(X.double(), W),
    lambda: causal_conv1d(X, W, None, "none", torch.zeros(2, 4, 16)),
    lambda: causal_conv1d(X, W, None, "none", torch.zeros(2, 3, 16).half()),
    lambda: causal_conv1d_step(X, torch.zeros(2, 3, 16), W),
    lambda: causal_conv1d_step(X[:, 0], torch.zeros(2, 3, 16), W, None, "none", torch.zeros(2, 3, 8)),
    lambda: causal_conv1d_step(X[:, 0], torch.zeros(2, 16, 3).transpose(1, 2), W),
    lambda: selective_scan(X[0], X[0], A, ROWS[0], ROWS[0]),
    lambda: selective_scan(X, X[:, :4], A, ROWS, ROWS),
    lambda: selective_scan(X, X.half(), A, ROWS, ROWS),
    lambda: selective_scan(X, X, A[:8], ROWS, ROWS),
    lambda: selective_scan(X, X, torch.ones(16, 33), torch.zeros(2, 5, 33), torch.zeros(2, 5, 33)),
    lambda: selective_scan(X, X, A[:, :0], ROWS[..., :0], ROWS[..., :0]),
    lambda: selective_scan(X, X, A, ROWS[..., :2], ROWS),
    lambda: selective_scan(X, X, A, ROWS, ROWS, torch.ones(8)),
    lambda: selective_scan(X, X, A, ROWS, ROWS, None, X[..., :8]),
    lambda: selective_scan(X, X, A, ROWS, ROWS, None, None, torch.ones(16, 1)),
    lambda: selective_scan(X, X, A, ROWS, ROWS, initial_state=torch.zeros(2, 3, 16)),
    lambda: selective_scan(X, X, A, ROWS, ROWS, initial_state=torch.zeros(2, 16, 3).half()),
    lambda: selective_scan_step(X[:, 0], torch.zeros(2, 16, 3), X[:, 0], A, ROWS, ROWS),
    lambda: selective_scan_step(X[:, 0], torch.zeros(1, 16, 3).expand(2, 16, 3), X[:, 0], A, ROWS[:, 0], ROWS[:, 0]),
    lambda: rotary(Q[0], Q[0], POSITIONS, FREQUENCIES),
    lambda: rotary(Q, Q[:, :4], POSITIONS, FREQUENCIES),
    lambda: rotary(Q, Q.half(), POSITIONS, FREQUENCIES),
    lambda: rotary(Q[..., :20], Q[..., :20], POSITIONS, FREQUENCIES[:8]),
    lambda: rotary(Q, Q, POSITIONS[:4], FREQUENCIES),
    lambda: rotary(Q, Q, POSITIONS.half(), FREQUENCIES),
    lambda: rotary(Q, Q, POSITIONS, FREQUENCIES.float()),
    lambda: rotary(Q, Q, POSITIONS, FREQUENCIES[:4]),
    lambda: rotary(Q, Q, POSITIONS, rotary_frequencies(48)),
    lambda: rotary(Q, Q, POSITIONS, FREQUENCIES, scale=float("nan")),
    lambda: head_norm_rotary(Q, Q, torch.ones(32), None, POSITIONS, FREQUENCIES),
    lambda: head_norm_rotary(Q, Q, torch.ones(32), torch.ones(16), POSITIONS, FREQUENCIES),
    lambda: head_norm_rotary(Q, Q, torch.ones(32), torch.ones(32), POSITIONS, FREQUENCIES, eps=-1.0),
])  # fmt: skip
def test_bad_arguments_are_refused(call):
    with pytest.raises(AssertionError):
        call()


def test_states_have_no_gradients():
    with pytest.raises(RuntimeError, match="detach"):
        causal_conv1d(X, W, None, "none", torch.zeros(2, 3, 16, requires_grad=True))
    with pytest.raises(RuntimeError, match="detach"):
        selective_scan(X, X, A, ROWS, ROWS, initial_state=torch.zeros(2, 16, 3, requires_grad=True))
    with pytest.raises(RuntimeError, match="detach"):
        selective_scan_step(X[:, 0], torch.zeros(2, 16, 3, requires_grad=True), X[:, 0], A, ROWS[:, 0], ROWS[:, 0])


def test_states_that_overlap_are_refused():
    flat = torch.zeros(400)
    with pytest.raises(AssertionError, match="overlaps state"):
        causal_conv1d_step(X[:, 0], flat[:96].view(2, 3, 16), W, out_state=flat[48:144].view(2, 3, 16))
    with pytest.raises(AssertionError, match="overlaps an input"):
        causal_conv1d_step(flat[:48].view(3, 16)[:2], flat[:96].view(2, 3, 16), W)
    with pytest.raises(AssertionError, match="overlaps an input"):  # a state within the rows of a wider tensor
        selective_scan_step(flat[:64].view(2, 32)[:, :16], flat[16:112].view(2, 16, 3), X[:, 0], A, ROWS[:, 0], ROWS[:, 0])
    a = torch.zeros(4, 4)
    assert overlap(a, a) and overlap(a[:, 0], a[:, 1]) and not overlap(a[:2], a[2:]) and not overlap(a, a[:0])


def test_layers_refuse_what_the_kernels_do_not_take():
    for call in (
        lambda: CausalConv1d(12, 4), lambda: CausalConv1d(16, 1), lambda: CausalConv1d(16, 9),
        lambda: CausalConv1d(16, 4, activation="gelu"), lambda: SelectiveScan(0), lambda: SelectiveScan(16, 33),
        lambda: SelectiveScan(16, 4, 0.1, 0.01), lambda: HeadNormRotary(64, rotated=3), lambda: HeadNormRotary(64, method="other"),
    ):  # fmt: skip
        with pytest.raises(ValueError):
            call()
    assert SelectiveScan(16, 4).empty_state(3).shape == (3, 16, 4)
    assert CausalConv1d(16, 4).empty_state(3).shape == (3, 3, 16)
    layer = HeadNormRotary(64).half()
    assert layer.q_weight.dtype == torch.float16 and layer.frequencies.dtype == torch.float64
    assert "frequencies" not in layer.state_dict()
    steps = torch.nn.functional.softplus(SelectiveScan(1000).delta_bias)
    assert 0.9e-3 < steps.min() < 2e-3 and 0.05 < steps.max() < 0.11


def test_meta_tensors():
    x, w = X.to("meta"), W.to("meta")
    y, state = causal_conv1d_forward(x, w, None, "silu", None, True)
    assert y.shape == (2, 5, 16) and state.shape == (2, 3, 16)
    y, state, kept = selective_scan_forward(x, x, A.to("meta"), ROWS.to("meta"), ROWS.to("meta"), None, None, None, True, None, True, True)
    assert y.shape == (2, 5, 16) and state.shape == (2, 16, 3) and kept.shape == (2, 1, 3, 16) and state.dtype == torch.float32


def test_rows_of():
    wide = torch.zeros(3, 7, 40)
    for t, row in ((wide, 40), (wide[..., :16], 40), (wide[..., 3:5], 40), (wide[:1, :, :16], 40), (wide[:, :1, :16], 280),
                   (wide[:1, :1], 40), (wide[:, 0], 280), (wide[..., :1], 40)):  # fmt: skip
        got, distance = rows_of(t)
        assert got.data_ptr() == t.data_ptr() and distance == row, (t.shape, t.stride())
    for t in (wide[:, :6], wide[..., ::2], wide.transpose(0, 1), wide[:, :, :1].expand(3, 7, 4), torch.zeros(3, 1, 4).expand(3, 7, 4)):
        got, distance = rows_of(t)
        assert got.is_contiguous() and distance == t.shape[-1] and torch.equal(got, t)
    assert rows_of(None) == (None, 0)
    assert rows_of(wide[..., :16], 8)[0].data_ptr() == wide.data_ptr()
    for t in (wide[..., 2:18], torch.zeros(3, 7, 18)[..., :16]):  # rows that do not start on 16 bytes
        assert rows_of(t, 8)[0].data_ptr() != t.data_ptr()
    far = torch.empty((1 << 26) + 16, dtype=torch.float16)  # eight rows of which pass 31 bits
    for row, copied in (((1 << 26) - 8, False), (1 << 26, True)):
        t = far.as_strided((1, 2, 16), (0, row, 1))
        assert (rows_of(t)[0].data_ptr() != t.data_ptr()) == copied and rows_of(t, 8)[1] == row


def test_frequencies_have_no_gradients():
    leaf = FREQUENCIES.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="frequencies"):
        rotary(Q, Q, POSITIONS, leaf)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU only"):
        rotary(Q, Q, POSITIONS, leaf)


def test_heads_of():
    rows = torch.zeros(2, 5, 6, 16)
    for t, distances in ((rows, (96, 16)), (rows[:, :, 1:3], (96, 16)), (rows[..., :8], (96, 16)), (rows[:1], (96, 16)),
                         (rows[:, :1], (480, 16)), (rows.transpose(1, 2)[:1], (16, 96))):  # fmt: skip
        got, row, head = _heads_of(t)
        assert got.data_ptr() == t.data_ptr() and (row, head) == distances
    for t in (rows[:, :4], rows[..., 1:9], rows[..., ::2], torch.zeros(2, 5, 6, 10)[..., :8]):
        got, row, head = _heads_of(t)
        assert got.is_contiguous() and (row, head) == (t.shape[2] * t.shape[3], t.shape[3])


def test_structures():
    assert fields_of("SpioConv1dArgs")[:3] == (("pointer", "x"), ("pointer", "weight"), ("pointer", "bias"))
    assert fields_of("SpioRotaryArgs")[-2:] == (("double", "eps"), ("double", "scale"))
    with open(os.path.join(CSRC_DIR, "spio_token_args.h"), encoding="utf-8") as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    for name in ("SpioScanArgs", "SpioConv1dArgs", "SpioRotaryArgs"):
        body = re.search(name + r" \{(.*?)\}", text, re.DOTALL).group(1)
        assert len(fields_of(name)) == body.count(",") + body.count(";")
    t = torch.zeros(4)
    filled = Arguments("SpioRotaryArgs", q=t, tokens=-1, scale=1.5)
    names = [f for _, f in fields_of("SpioRotaryArgs")]
    assert filled.array[names.index("q")] == t.data_ptr() and filled.array[names.index("k")] == 0
    assert filled.array[names.index("tokens")] == 2**64 - 1 and filled.array[names.index("scale")] == 0x3FF8 << 48
    for bad in (dict(nothing=1), dict(q=1), dict(tokens=t)):
        with pytest.raises(AssertionError):
            Arguments("SpioRotaryArgs", **bad)


def test_work_is_cut_alike_on_both_paths():
    """The native call path computes what kernels/*_kernel.py do."""
    other = native._native
    if other is None:
        pytest.skip("no native call path")
    sizes = [1, 2, 3, 7, 16, 47, 48, 49, 100, 777, 4099, 100000]
    for tokens in sizes:
        for sequences in (1, 2, 9, 128, 5000):
            for channels in (8, 64, 72, 768, 4096):
                for backward in (False, True):
                    assert other.scan_chunk(tokens, channels, sequences, backward) == chunk_tokens(tokens, channels, sequences, backward)
                    assert other.conv1d_slice(tokens, channels, sequences, backward) == slice_tokens(tokens, channels, sequences, backward)
        for heads in (1, 2, 9, 64):
            for head, norm in ((h, norm) for h in (8, 32, 80, 128, 256) for norm in (False, True)):
                parts = parts_of(tokens, heads, head, norm)
                assert other.rotary_parts(tokens, heads, head, norm) == parts and 1 <= parts <= heads
                for summed in (False, True):
                    assert other.rotary_grid(tokens, parts, head, norm, summed) == grid_of(tokens, parts, head, norm, summed)
    for states in range(1, 33):
        assert other.scan_tile(states) == tile_tokens(states)


def test_chunks_and_slices_cover_the_tokens():
    for tokens in (1, 15, 16, 33, 196, 2048, 4099):
        for channels, sequences in ((1, 1), (64, 2), (1536, 1), (2048, 4), (768, 128), (4096, 64)):
            for backward in (False, True):
                chunk = chunk_tokens(tokens, channels, sequences, backward)
                waves = -(-channels // 64) * sequences
                assert chunk >= min(tokens, 16)
                assert chunk >= tokens or chunk % 8 == 0  # whole tiles
                assert -(-tokens // chunk) * waves <= max(4096, waves)
    assert all(8 % tile_tokens(states) == 0 for states in range(1, 33))
    assert [lanes_of(d, True) for d in (8, 16, 24, 32, 64, 80, 128, 136, 256)] == [1, 1, 2, 2, 4, 8, 8, 16, 16]
    assert [lanes_of(d, False) for d in (8, 16, 24, 32, 64, 80, 128, 136, 256)] == [1, 1, 2, 2, 4, 5, 8, 9, 16]


def test_frequencies():
    plain = rotary_frequencies(64)
    assert plain.dtype == torch.float64 and plain.shape == (32,)
    torch.testing.assert_close(plain, torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64))
    assert torch.equal(rotary_frequencies(64, factor=1.0, method="ramp"), plain)
    torch.testing.assert_close(rotary_frequencies(64, factor=8.0), plain / 8)
    stretched = rotary_frequencies(64, factor=8.0, method="base")
    assert stretched[0] == 1 and math.isclose(stretched[-1], plain[-1] / 8, rel_tol=1e-12)
    ramp = rotary_frequencies(64, factor=8.0, method="ramp", trained_tokens=4096)
    turns = plain * 4096 / (2 * math.pi)
    assert torch.equal(ramp[turns >= 32], plain[turns >= 32])
    torch.testing.assert_close(ramp[turns <= 1], plain[turns <= 1] / 8)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (ramp[between] < plain[between]).all() and (ramp[between] > plain[between] / 8).all()
    assert (ramp[1:] < ramp[:-1]).all()
    assert rotary_frequencies(2, base=500.0, factor=2.0, method="base").tolist() == [1.0]
    for bad in (dict(channels=0), dict(channels=7), dict(channels=8, base=1.0), dict(channels=8, factor=0.5),
                dict(channels=8, method="x"), dict(channels=8, method="ramp", slow_turns=4.0, fast_turns=4.0)):  # fmt: skip
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


WIDE_SHIFT = re.compile(r"v_(?:lshl|lshr|ashr)rev_[bi]64\S* v\[\d+:\d+\], v\d+")
PACKED = re.compile(r"v_pk_(?:add|mul|fma)_f32")
SCAN = kernels.SelectiveScanParams
COMPILED = [
    (kernels.causal_conv1d_kernel_factory, kernels.CausalConv1dParams(4, 1, 2, 2)),
    (kernels.causal_conv1d_bwd_kernel_factory, kernels.CausalConv1dParams(4, 1, 2, 2)),
    (kernels.causal_conv1d_bwd_kernel_factory, kernels.CausalConv1dParams(8, 2, 2, 2)),
    (kernels.causal_conv1d_sums_kernel_factory, kernels.CausalConv1dParams(4, 1, 2, 2)),
    (kernels.causal_conv1d_step_kernel_factory, kernels.CausalConv1dParams(4, 0, 0, 2)),
    (kernels.selective_scan_ends_kernel_factory, SCAN(16, 1, False, True)),
    (kernels.selective_scan_kernel_factory, SCAN(16, 1, True, True, True)),
    (kernels.selective_scan_ends_bwd_kernel_factory, SCAN(16, 1, True, True)),
    (kernels.selective_scan_bwd_kernel_factory, SCAN(16, 1, True, True)),
    (kernels.selective_scan_bwd_kernel_factory, SCAN(15, 0, True, True)),
    (kernels.selective_scan_bwd_kernel_factory, SCAN(8, 2, True, True)),
    (kernels.selective_scan_bwd_kernel_factory, SCAN(32, 2, True, True)),
    (kernels.selective_scan_sums_kernel_factory, SCAN(16, 1)),
    (kernels.selective_scan_join_kernel_factory, SCAN(16, 1)),
    (kernels.selective_scan_step_kernel_factory, SCAN(16, 1, True, True)),
    (kernels.head_norm_rotary_kernel_factory, kernels.HeadNormRotaryParams(128, 1)),
    (kernels.head_norm_rotary_bwd_kernel_factory, kernels.HeadNormRotaryParams(128, 1)),
    (kernels.head_norm_rotary_bwd_kernel_factory, kernels.HeadNormRotaryParams(256, 2, True, True)),
]


@pytest.mark.parametrize("factory,params", COMPILED, ids=lambda v: v.encode() if hasattr(v, "encode") else v.get_kernel_name())
def test_compiled_code(factory, params, tmp_path):
    """No 64-bit shift by a vector register, no packed float32, no registers kept in memory."""
    kernel = factory.make_kernel(params, factory.configs(params, DeviceAttributes())[0], DeviceAttributes())
    out = str(tmp_path / "kernel.s")
    subprocess.run([os.path.join(ROCM_HOME, "bin", "hipcc"), "-S", "--cuda-device-only", *HIPCC_DEVICE_FLAGS, f"-I{CSRC_DIR}",
                    *[f"-D{k}={v}" for k, v in kernel.defines.items()], "-o", out,
                    os.path.join(CSRC_DIR, kernel.kernel_source_file)], check=True, capture_output=True)  # fmt: skip
    with open(out, encoding="utf-8") as f:
        code = f.read()
    assert "s_endpgm" in code and not WIDE_SHIFT.findall(code) and not PACKED.findall(code)
    assert int(re.search(r"\.private_segment_fixed_size:\s+(\d+)", code).group(1)) == 0
