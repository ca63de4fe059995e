"""The operators over sequences of tokens as a model uses them: layers of both kinds one after the other, trained and
served token by token; on another stream; timed launch by launch."""

import pytest
import torch
from torch import nn

from spio_amd.functional import selective_scan
from spio_amd.kernels.kernel import LaunchTimer
from spio_amd.layers import CausalConv1d, HeadNormRotary, SelectiveScan

pytestmark = pytest.mark.gpu


class StateSpaceLayer(nn.Module):
    def __init__(self, width, inner, states, rank):
        super().__init__()
        self.inner, self.states, self.rank = inner, states, rank
        self.into = nn.Linear(width, 2 * inner, bias=False)
        self.conv = CausalConv1d(inner, 4, activation="silu")
        self.project = nn.Linear(inner, rank + 2 * states, bias=False)
        self.step_up = nn.Linear(rank, inner, bias=False)
        self.scan = SelectiveScan(inner, states)
        self.out = nn.Linear(inner, width, bias=False)

    def _rows(self, x):
        delta, B, C = self.project(x).split([self.rank, self.states, self.states], -1)
        return self.step_up(delta), B, C

    def forward(self, x, return_state=False):
        x, gate = self.into(x).chunk(2, -1)  # parts of wider rows
        if not return_state:
            x = self.conv(x)
            return self.out(self.scan(x, *self._rows(x), gate))
        x, conv_state = self.conv(x, return_state=True)
        y, state = self.scan(x, *self._rows(x), gate, return_state=True)
        return self.out(y), (conv_state, state)

    def step(self, x, states):
        x, gate = self.into(x).chunk(2, -1)
        x = self.conv.step(x, states[0])
        delta, B, C = self._rows(x)
        return self.out(self.scan.step(x, states[1], delta, B, C, gate))


class AttentionLayer(nn.Module):
    def __init__(self, width, heads, shared):
        super().__init__()
        self.heads, self.shared, self.d = heads, shared, width // heads
        self.qkv = nn.Linear(width, (heads + 2 * shared) * self.d, bias=False)
        self.norm = HeadNormRotary(self.d, rotated=self.d // 2, interleaved=True)
        self.out = nn.Linear(width, width, bias=False)

    def forward(self, x, cache=None, first=0):
        rows = self.qkv(x).unflatten(-1, (-1, self.d))
        q, k, v = rows.split([self.heads, self.shared, self.shared], 2)
        q, k = self.norm(q, k, torch.arange(x.shape[1], device=x.device) + first)
        if cache is not None:
            k, v = torch.cat([cache[0], k], 1), torch.cat([cache[1], v], 1)
        with torch.autocast("cuda", enabled=False):  # products over batches in float32, of operands without gaps
            group = self.heads // self.shared
            qf = q.float().transpose(1, 2).contiguous()
            kf, vf = (t.float().repeat_interleave(group, 2).transpose(1, 2) for t in (k, v))
            scores = qf @ kf.transpose(-1, -2).contiguous() * self.d**-0.5
            after = torch.arange(k.shape[1], device=x.device) > torch.arange(x.shape[1], device=x.device)[:, None] + first
            y = (scores.masked_fill(after, float("-inf")).softmax(-1) @ vf.contiguous()).transpose(1, 2).to(q.dtype)
        return self.out(y.flatten(-2)), (k, v)


def _model():
    torch.manual_seed(0)
    return StateSpaceLayer(64, 128, 16, 4).cuda(), AttentionLayer(64, 4, 2).cuda()


def test_trained():
    """All parameters of both layers get gradients; a differing token changes nothing before it."""
    mixer, attention = _model()
    x = torch.randn(2, 50, 64, device="cuda", requires_grad=True)
    y = attention(x + mixer(x))[0]
    y.square().mean().backward()
    for p in (*mixer.parameters(), *attention.parameters(), x):
        assert p.grad is not None and p.grad.isfinite().all() and p.grad.any()
    with torch.no_grad():
        other = x.detach().clone()
        other[:, 30] += 1
        z = attention(other + mixer(other))[0]
    torch.testing.assert_close(z[:, :30], y.detach()[:, :30], rtol=1e-4, atol=1e-5)
    assert ((z - y.detach())[:, 30:].abs() > 1e-4).any()


def test_gradient_along_a_direction():
    """The whole model's gradient for its inputs against differences of the loss, in float32."""
    mixer, attention = _model()
    x = torch.randn(1, 40, 64, device="cuda", requires_grad=True)
    dy = torch.randn(1, 40, 64, device="cuda")

    def loss(x):
        return (attention(x + mixer(x))[0] * dy).double().sum()

    (dx,) = torch.autograd.grad(loss(x), x)
    direction = dx / dx.norm()
    with torch.no_grad():
        slope = (loss(x + 0.01 * direction) - loss(x - 0.01 * direction)) / 0.02
    # a loss of magnitude 30 is off by 1e-5, over 0.02; the third derivative along a unit direction times 1.7e-5
    assert abs(float(slope) - float(dx.norm())) <= 2e-3 * float(dx.norm()) + 1e-3


def test_served():
    """A prompt, then token by token, gives what the whole sequence at once gives."""
    mixer, attention = _model()
    x = torch.randn(2, 24, 64, device="cuda")
    with torch.no_grad():
        whole = attention(x + mixer(x))[0]
        y, states = mixer(x[:, :20], return_state=True)
        out, cache = attention(x[:, :20] + y)
        rows = [out]
        for t in range(20, 24):
            h = x[:, t] + mixer.step(x[:, t], states)
            out, cache = attention(h[:, None], cache, t)
            rows.append(out)
    torch.testing.assert_close(torch.cat(rows, 1), whole, rtol=1e-4, atol=1e-4)


def test_under_autocast():
    mixer, attention = _model()
    x = torch.randn(2, 20, 64, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = mixer(x)
        z, _ = attention(y)
    assert y.dtype == z.dtype == torch.bfloat16
    z.float().sum().backward()
    assert all(p.grad.dtype == torch.float32 and p.grad.isfinite().all() for p in mixer.parameters())


def _scan_inputs(seed, n=2, l=100, c=70, s=16):
    g = torch.Generator().manual_seed(seed)
    rows = lambda *shape: torch.randn(*shape, generator=g).cuda()  # noqa: E731
    return rows(n, l, c), rows(n, l, c), -rows(c, s).abs(), rows(n, l, s), rows(n, l, s)


def test_streams():
    """Two streams at once, each behind work of its own, with workspaces of their own."""
    expected = [selective_scan(*_scan_inputs(i), delta_softplus=True) for i in range(2)]
    inputs = [_scan_inputs(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    a = torch.randn(2048, 2048, device="cuda")
    got = []
    for stream, args in zip(streams, inputs):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            b = a
            for _ in range(10):
                b = b @ a * 1e-3
            late = args[0] + b[0, 0] * 0
            got.append(selective_scan(late, *args[1:], delta_softplus=True))
    for stream in streams:
        stream.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, expected))


def test_two_graphs_in_one_pool():
    """Two captured scans that share a memory pool, replayed in the order of their capture."""
    static = [_scan_inputs(i) for i in range(2)]
    expected = [selective_scan(*args, delta_softplus=True) for args in static]
    torch.cuda.synchronize()
    graphs, out, pool = [], [], None
    for args in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out.append(selective_scan(*args, delta_softplus=True))
        pool = graph.pool()
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, expected))


def test_launches_are_timed():
    args = _scan_inputs(0)
    with LaunchTimer() as timer:
        selective_scan(*args, delta_softplus=True)
    names = sorted(k.kernel_name.split("__")[0] for k in timer.averages())
    assert names == ["spio_selective_scan", "spio_selective_scan_ends", "spio_selective_scan_join"]
