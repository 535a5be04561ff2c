"""Each dense and state-space entry point as the first call of a fresh process,
inside a graph capture, and two graphs of one call replayed in turn: the bits of
the eager call."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

CODE = """
import torch
from ervf_b200 import GPUKernels
dev = torch.device("cuda", 0)
g = torch.Generator(device=dev).manual_seed(0)
rnd = lambda *s: torch.randn(*s, generator=g, device=dev)
k = GPUKernels()
h, p, gr, n, w, t = 6, 64, 2, 128, 4, 300
inner, ch = h * p, h * p + 2 * gr * n
W, x = rnd(384, 256).bfloat16(), rnd(t, 256).bfloat16()
xbc, dt, z = rnd(t, ch).bfloat16(), rnd(t, h).bfloat16(), rnd(t, inner).bfloat16()
cw, cb, nw = rnd(ch, w), rnd(ch), rnd(inner)
A, D, bias = -rnd(h).abs(), rnd(h), rnd(h) - 3
cu = torch.tensor([0, 100, t], dtype=torch.int32, device=dev)
zero = lambda *s, d=torch.bfloat16: torch.zeros(*s, dtype=d, device=dev)
conv0, ssm0 = rnd(2, w - 1, ch).bfloat16(), rnd(2, h, p, n)
has = torch.tensor([True, True], device=dev)

def linear(o, m):
    k.linear_bf16(o, W, x[:m], 384, 256, m)
def conv(o, s):
    k.conv1d_prompt(o, xbc, cw, cb, s, cu, 2, t, ch, w, has_state=has)
def scan(o, s):
    k.ssm_prompt(o, xbc[:, :inner], dt, A, xbc[:, inner:inner + gr * n], xbc[:, inner + gr * n:], D, bias, s, cu, 2, t,
                 h, p, gr, n, has_state=has)
def token(o, c, s):
    k.ssm_token(o, xbc[:2], dt[:2], cw, cb, c, A, D, bias, s, 2, h, p, gr, n, w, z=z[:2], norm_w=nw)
def norm(o):
    k.gated_norm(o, z, z, nw, t, gr, inner // gr)

calls = {
    "linear_one": (lambda b: linear(b[0], 1), lambda: [zero(1, 384)]),
    "linear_some": (lambda b: linear(b[0], 60), lambda: [zero(60, 384)]),
    "linear_many": (lambda b: linear(b[0], t), lambda: [zero(t, 384)]),
    "conv": (lambda b: conv(*b), lambda: [zero(t, ch), conv0.clone()]),
    "scan": (lambda b: scan(*b), lambda: [zero(t, inner), ssm0.clone()]),
    "token": (lambda b: token(*b), lambda: [zero(2, inner), conv0.clone(), ssm0.clone()]),
    "norm": (lambda b: norm(b[0]), lambda: [zero(t, inner)]),
}
for name, (call, make) in calls.items():
    graphs = []
    for _ in range(2):
        bufs = make()
        start = [b.clone() for b in bufs]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(bufs)
        graphs.append((graph, bufs, start))
    eager = make()
    call(eager)
    for _ in range(2):
        for graph, bufs, start in graphs:
            for b, s in zip(bufs, start):
                b.copy_(s)
            graph.replay()
    torch.cuda.synchronize()
    for _, bufs, _ in graphs:
        for b, e in zip(bufs, eager):
            assert torch.equal(b, e), name
print("graphs ok")
"""


def test_first_call_inside_a_capture(cuda):
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "graphs ok" in r.stdout, r.stdout[-1500:] + r.stderr[-3000:]
