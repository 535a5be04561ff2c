"""The dense projection with its epilogue against 64 bits.

Tolerance: bf16 products are exact in f32; a sum of `cols` of them in any
order is off by at most cols * 2^-23 of the sum of their magnitudes (a step
that truncates instead of rounding loses a whole unit in the last place), the
epilogue's operations by a few 2^-24 of their values, the output by half a
step of its type."""

from __future__ import annotations

import pytest
import torch

import hybrid_ref as ref

pytestmark = pytest.mark.gpu


def bound(out, size, cols, dtype):
    return ref.HALF[dtype] * out.abs() + (2 * cols + 32) * ref.U * size + 1e-30


def make(rows, cols, tokens, dtype, bias, resid, seed=0):
    g = torch.Generator().manual_seed(seed)
    W = (torch.randn(rows, cols, generator=g) * 0.1).bfloat16()
    x = torch.randn(tokens, cols, generator=g).bfloat16()
    b = torch.randn(rows, generator=g) if bias else None
    r = torch.randn(tokens, rows, generator=g).to(dtype) if resid else None
    return W, x, b, r


def put(v, dev):
    return None if v is None else v.to(dev)


@pytest.fixture(scope="module")
def k(cuda):
    from ervf_b200 import GPUKernels

    return GPUKernels()


@pytest.mark.parametrize("rows,cols,tokens", [
    (1, 8, 1), (7, 16, 3), (128, 64, 1), (129, 72, 33), (300, 1000, 17), (256, 4104, 2),
    (1000, 264, 128), (257, 520, 129), (513, 136, 300), (2688, 4096, 1), (2688, 1856, 8),
    (640, 328, 257), (1111, 88, 511), (20000, 64, 5), (96, 8192, 64),
    (2500, 200, 2001), (5000, 72, 1030), (300, 1032, 9000), (2700, 136, 3333)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear(k, cuda, rows, cols, tokens, dtype):
    W, x, b, r = make(rows, cols, tokens, dtype, True, True)
    out = torch.full((tokens, rows), float("nan"), dtype=dtype, device=cuda)
    k.linear_bf16(out, put(W, cuda), put(x, cuda), rows, cols, tokens, bias=put(b, cuda), act="silu",
                  resid=put(r, cuda))
    want, size = ref.linear(W, x, b, "silu", r)
    ref.within(out, want, bound(want, size, cols, dtype))


@pytest.mark.parametrize("rows,cols,tokens", [
    (2688, 4096, 100), (1111, 2056, 129),        # 128 x 128, a tile's columns shared
    (8000, 200, 300),                            # not shared
    (3700, 2696, 380), (10000, 1000, 300),       # 128 x 256, shared and not
    (2600, 2200, 401), (3712, 2688, 512),        # pairs, shared
    (3700, 1400, 1000), (5000, 1400, 3001)])     # one and several tiles each
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tiles(k, cuda, rows, cols, tokens, dtype):
    W, x, b, r = make(rows, cols, tokens, dtype, True, True, seed=6)
    out = torch.full((tokens, rows), float("nan"), dtype=dtype, device=cuda)
    k.linear_bf16(out, put(W, cuda), put(x, cuda), rows, cols, tokens, bias=put(b, cuda), act="relu2",
                  resid=put(r, cuda))
    want, size = ref.linear(W, x, b, "relu2", r)
    ref.within(out, want, bound(want, size, cols, dtype))


@pytest.mark.parametrize("act", ["none", "relu2", "silu", "gelu"])
@pytest.mark.parametrize("bias,resid", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("tokens", [3, 140])
def test_epilogue(k, cuda, act, bias, resid, tokens):
    W, x, b, r = make(200, 96, tokens, torch.float32, bias, resid, seed=1)
    out = torch.empty(tokens, 200, device=cuda)
    k.linear_bf16(out, put(W, cuda), put(x, cuda), 200, 96, tokens, bias=put(b, cuda), act=act, resid=put(r, cuda))
    want, size = ref.linear(W, x, b, act, r)
    ref.within(out, want, bound(want, size, 96, torch.float32))


@pytest.mark.parametrize("tokens", [5, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_guards_and_residual_in_place(k, cuda, tokens, dtype):
    """x and out are slices of wider rows; the bytes beside them stay as they were; resid is out."""
    rows, cols = 331, 136
    W, x, b, r = make(rows, cols, tokens, dtype, True, True, seed=2)
    wide_x = torch.full((tokens, 200), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide_x[:, 32:32 + cols] = x.to(cuda)
    wide = torch.full((tokens + 1, 400), 7.0, dtype=dtype, device=cuda)
    view = wide[:tokens, 3:3 + rows]
    view.copy_(r)
    k.linear_bf16(view, put(W, cuda), wide_x[:, 32:32 + cols], rows, cols, tokens, bias=put(b, cuda), resid=view)
    want, size = ref.linear(W, x, b, "none", r)
    ref.within(view, want, bound(want, size, cols, dtype))
    assert (wide[:, :3] == 7).all() and (wide[:, 3 + rows:] == 7).all() and (wide[tokens] == 7).all()


@pytest.mark.parametrize("rows,cols,tokens", [(331, 136, 200), (334, 1048, 70), (2699, 2696, 381), (3705, 1400, 1001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_aligned_rows_that_end_inside_a_tile(k, cuda, rows, cols, tokens, dtype):
    """Rows on 16-byte boundaries, neither rows nor tokens whole tiles: what lies beside them stays."""
    W, x, b, r = make(rows, cols, tokens, dtype, True, True, seed=7)
    wide = torch.full((tokens + 40, rows // 8 * 8 + 64), 7.0, dtype=dtype, device=cuda)
    view = wide[:tokens, 8:8 + rows]
    view.copy_(r)
    k.linear_bf16(view, put(W, cuda), put(x, cuda), rows, cols, tokens, bias=put(b, cuda), act="silu", resid=view)
    want, size = ref.linear(W, x, b, "silu", r)
    ref.within(view, want, bound(want, size, cols, dtype))
    assert (wide[:, :8] == 7).all() and (wide[:, 8 + rows:] == 7).all() and (wide[tokens:] == 7).all()


@pytest.mark.parametrize("rows,cols,tokens", [
    (331, 1048, 70), (8001, 200, 300), (3699, 2696, 380), (10001, 1000, 300), (2599, 2200, 401), (3699, 1400, 1001)])
def test_rows_of_any_alignment_in_every_tile(k, cuda, rows, cols, tokens):
    W, x, b, r = make(rows, cols, tokens, torch.bfloat16, True, True, seed=9)
    wide = torch.full((tokens + 1, rows + 10), 7.0, dtype=torch.bfloat16, device=cuda)
    view = wide[:tokens, 3:3 + rows]
    k.linear_bf16(view, put(W, cuda), put(x, cuda), rows, cols, tokens, bias=put(b, cuda), act="gelu",
                  resid=put(r, cuda))
    want, size = ref.linear(W, x, b, "gelu", r)
    ref.within(view, want, bound(want, size, cols, torch.bfloat16))
    assert (wide[:, :3] == 7).all() and (wide[:, 3 + rows:] == 7).all() and (wide[tokens] == 7).all()


@pytest.mark.parametrize("tokens", [1, 40, 200])
def test_same_bits_every_call(k, cuda, tokens):
    W, x, _, _ = make(2688, 4096, tokens, torch.float32, False, False, seed=3)
    W, x = W.to(cuda), x.to(cuda)
    outs = [torch.empty(tokens, 2688, device=cuda) for _ in range(3)]
    for o in outs:
        k.linear_bf16(o, W, x, 2688, 4096, tokens)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_infinities_stay_in_their_rows(k, cuda):
    W, x, _, _ = make(130, 64, 150, torch.float32, False, False, seed=4)
    x[17, 5], x[140, 9] = float("inf"), float("nan")
    out = torch.empty(150, 130, device=cuda)
    k.linear_bf16(out, put(W, cuda), put(x, cuda), 130, 64, 150, act="relu2")
    clean = torch.isfinite(out).all(1).cpu()
    assert [int(v) for v in (~clean).nonzero().flatten()] == [17, 140]
    assert torch.isnan(out[140]).all()


@pytest.mark.parametrize("tokens", [5, 150, 700])
def test_bias_of_any_alignment(k, cuda, tokens):
    W, x, b, _ = make(1024, 512, tokens, torch.float32, True, False, seed=10)
    shifted = torch.cat([torch.zeros(1), b]).to(cuda)[1:]
    out = torch.empty(tokens, 1024, device=cuda)
    k.linear_bf16(out, put(W, cuda), put(x, cuda), 1024, 512, tokens, bias=shifted)
    want, size = ref.linear(W, x, b, "none", None)
    ref.within(out, want, bound(want, size, 512, torch.float32))


def test_no_tokens(k, cuda):
    W = torch.zeros(16, 16, dtype=torch.bfloat16, device=cuda)
    k.linear_bf16(torch.empty(0, 16, device=cuda), W, torch.empty(0, 16, dtype=torch.bfloat16, device=cuda), 16, 16, 0)


def test_captured_and_replayed(k, cuda):
    W, x, _, _ = make(384, 256, 70, torch.bfloat16, False, False, seed=5)
    W, x = W.to(cuda), x.to(cuda)
    out = torch.zeros(70, 384, dtype=torch.bfloat16, device=cuda)
    want = torch.empty_like(out)
    k.linear_bf16(want, W, x, 384, 256, 70)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        k.linear_bf16(out, W, x, 384, 256, 70)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    x.neg_()
    k.linear_bf16(want, W, x, 384, 256, 70)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_wrong_arrays_are_refused(k, cuda):
    W, x, _, _ = make(32, 64, 4, torch.float32, False, False)
    W, x, out = W.to(cuda), x.to(cuda), torch.zeros(4, 32, device=cuda)
    for bad in (dict(act="tanh"), dict(resid=torch.zeros(4, 32, device=cuda).bfloat16()),
                dict(bias=torch.zeros(31, device=cuda)), dict(bias=torch.zeros(32)), ):
        with pytest.raises(ValueError):
            k.linear_bf16(out, W, x, 32, 64, 4, **bad)
    with pytest.raises(ValueError):
        k.linear_bf16(out, W, x.float(), 32, 64, 4)
    with pytest.raises(ValueError):
        k.linear_bf16(out, W, x, 32, 64, 5)
    with pytest.raises(ValueError):
        k.linear_bf16(out, W, x[:, 1:], 32, 56, 4)       # not 16-byte aligned
    with pytest.raises(ValueError):
        k.linear_bf16(out.half(), W, x, 32, 64, 4)
    assert (out == 0).all()


def test_two_streams_and_a_graph_beside_them(k, cuda):
    """Calls of every tile form at once on two streams, and the same calls captured, give the bits
    of one after the other."""
    shapes = [(1200, 1160, 1), (2688, 2696, 100), (3700, 2696, 380), (2600, 2200, 401), (3700, 1400, 1000)]
    data = []
    for i, (rows, cols, tokens) in enumerate(shapes):
        W, x, b, r = (v.to(cuda) for v in make(rows, cols, tokens, torch.bfloat16, True, True, seed=20 + i))
        data.append((W, x, b, r, rows, cols, tokens))

    def run(which, outs):
        for i in which:
            W, x, b, r, rows, cols, tokens = data[i]
            k.linear_bf16(outs[i], W, x, rows, cols, tokens, bias=b, act="silu", resid=r)

    def fresh():
        return [torch.zeros(d[6], d[4], dtype=torch.bfloat16, device=cuda) for d in data]

    every = range(len(data))
    want, first, second, third = fresh(), fresh(), fresh(), fresh()
    run(every, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(every, third)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s):
            run(every, first)
            g.replay()
        with torch.cuda.stream(t):
            run(reversed(every), second)
    torch.cuda.synchronize()
    for i in every:
        assert torch.equal(want[i], first[i]) and torch.equal(want[i], second[i]) and torch.equal(want[i], third[i])
