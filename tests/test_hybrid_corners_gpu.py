"""Calls of the dense and state-space methods that their documentation allows, at the ends of their
ranges: few features for many tokens, one column block, arrays of more than 2^31 elements, outputs in
place of either input."""

from __future__ import annotations

import pytest
import torch

import hybrid_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16, U = torch.float32, torch.bfloat16, ref.U


@pytest.fixture(scope="module")
def k(cuda):
    from ervf_b200 import GPUKernels

    return GPUKernels()


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 7, 8, 9, 31, 33])
@pytest.mark.parametrize("tokens,cols", [(65, 8), (300, 72), (2000, 136)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_features_for_many_tokens(k, cuda, rows, tokens, cols, dtype):
    """In rows of their own width, and inside wider ones on 16-byte boundaries."""
    g = torch.Generator().manual_seed(rows)
    W, x = (torch.randn(n, cols, generator=g).bfloat16() for n in (rows, tokens))
    b, r = torch.randn(rows, generator=g), torch.randn(tokens, rows, generator=g).to(dtype)
    want, size = ref.linear(W, x, b, "silu", r)
    for wide in (rows, 64):
        out = torch.full((tokens + 1, wide), 7.0, dtype=dtype, device=cuda)
        out[:tokens, :rows] = r.to(cuda)
        k.linear_bf16(out[:tokens, :rows], W.to(cuda), x.to(cuda), rows, cols, tokens, bias=b.to(cuda), act="silu",
                      resid=out[:tokens, :rows])
        ref.within(out[:tokens, :rows], want, ref.HALF[dtype] * want.abs() + (2 * cols + 32) * U * size + 1e-30)
        assert (out[:, rows:] == 7).all() and (out[tokens] == 7).all()


@pytest.mark.parametrize("size,groups,shift", [(512, 2, 0), (512, 2, 1), (2000, 1, 0)])
@pytest.mark.parametrize("place", ["y", "z"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_in_place_of_either_input(k, cuda, size, groups, shift, place, dtype):
    g = torch.Generator().manual_seed(size)
    n = groups * size
    wide = [torch.randn(300, n + 8, generator=g).to(dtype) for _ in range(2)]
    y, z = (v.to(cuda)[:, shift:shift + n] for v in wide)
    w = torch.randn(n, generator=g)
    k.gated_norm(y if place == "y" else z, y, z, w.to(cuda), 300, groups, size)
    want, s = ref.gated_norm(*(v[:, shift:shift + n] for v in wide), w, groups, 1e-5)
    ref.within(y if place == "y" else z, want, ref.HALF[dtype] * want.abs() + (size / 2 + 32) * U * s + 1e-30)
    other = z if place == "y" else y
    assert torch.equal(other.cpu(), wide[1 if place == "y" else 0][:, shift:shift + n])


# ----------------------------------------------- more than 2^31 elements


@pytest.mark.parametrize("rows,tokens", [(131072, 16500), (600, 4_000_000), (72_000_000, 33)])
def test_projection_of_more_than_2_31_outputs(k, cuda, rows, tokens):
    g = torch.Generator(device=cuda).manual_seed(1)
    W, x = (torch.randn(n, 8, generator=g, device=cuda).bfloat16() for n in (rows, tokens))
    out = torch.full((tokens, rows), 9.0, dtype=BF16, device=cuda)
    k.linear_bf16(out, W, x, rows, 8, tokens)
    for t in (slice(0, 5), slice(tokens // 2, tokens // 2 + 5), slice(tokens - 5, tokens)):
        for r in (slice(0, 2000), slice(rows // 2 - 300, rows // 2), slice(max(0, rows - 2000), rows)):
            want, size = x[t].double() @ W[r].double().t(), x[t].double().abs() @ W[r].double().abs().t()
            assert ((out[t, r].double() - want).abs() <= 2.0**-8 * want.abs() + 48 * U * size).all()
    assert not (out == 9).all(1).any()


def test_packs_of_more_than_2_31_elements(k, cuda):
    """A long sequence and, behind 2^31 elements, a short one: this one's results are what they are
    alone (convolution and norm to the bit, the scan within its tolerance twice)."""
    h, p, gr, n, w = 64, 64, 8, 128, 4
    inner, ch, long, short = h * p, h * p + 2 * gr * n, 560_000, 200
    t = long + short
    g = torch.Generator(device=cuda).manual_seed(2)
    z = torch.empty(t, ch, dtype=BF16, device=cuda).normal_(generator=g)
    dt = torch.empty(t, h, dtype=BF16, device=cuda).normal_(generator=g)
    cu = torch.tensor([0, long, t], dtype=torch.int32, device=cuda)
    cw, cb = torch.randn(ch, w, generator=g, device=cuda), torch.randn(ch, generator=g, device=cuda)
    A, D, nw = -torch.rand(h, generator=g, device=cuda) - 1, torch.randn(h, generator=g, device=cuda), \
        torch.randn(inner, generator=g, device=cuda)

    def layer(z, dt, cu, seqs, t):
        conv = torch.zeros(seqs, w - 1, ch, dtype=BF16, device=cuda)
        state = torch.zeros(seqs, h, p, n, device=cuda)
        x = torch.empty_like(z)
        k.conv1d_prompt(x, z, cw, cb, conv, cu, seqs, t, ch, w)
        y = torch.empty(t, inner, dtype=BF16, device=cuda)
        k.ssm_prompt(y, x[:, :inner], dt, A, x[:, inner:inner + gr * n], x[:, inner + gr * n:], D, None, state, cu, seqs, t,
                     h, p, gr, n)
        return x, y, conv, state

    assert t * inner > 2**31 and t * ch > 2**31
    x, y, conv, state = layer(z, dt, cu, 2, t)
    x1, y1, conv1, state1 = layer(z[long:].contiguous(), dt[long:].contiguous(), None, 1, short)
    assert torch.equal(x[long:], x1) and torch.equal(conv[1], conv1[0])
    # the two cut the sequence at other places: both within the scan's tolerance
    _, size, _, state_size = ref.scan(
        *(v.cpu() for v in (x1[:, :inner].reshape(short, h, p), dt[long:], A, x1[:, inner:inner + gr * n].reshape(short, gr, n),
                            x1[:, inner + gr * n:].reshape(short, gr, n), D)), None, torch.zeros(1, h, p, n), [0, short], None,
        None)
    size = size.flatten(1).to(cuda)
    assert ((y[long:].double() - y1.double()).abs() <= 2 * (2.0**-8 * (y1.double().abs() + 2.0**-8 * size) +
                                                           (2.0**-8 + 1200 * U) * size)).all()
    assert ((state[1].double() - state1[0].double()).abs() <= 2 * 1200 * U * state_size[0].to(cuda) + 1e-30).all()
    del x
    before = y[-short:].clone()
    k.gated_norm(y, y, z[:, :inner], nw, t, gr, inner // gr)
    alone = torch.empty_like(before)
    k.gated_norm(alone, before, z[long:, :inner], nw, short, gr, inner // gr)
    assert torch.equal(y[long:], alone)


def test_one_token_step_of_slots_behind_2_31_elements(k, cuda):
    h, p, gr, n, w, slots = 64, 64, 8, 128, 4, 4200
    inner, ch = h * p, h * p + 2 * gr * n
    assert slots * inner * n > 2**31
    g = torch.Generator(device=cuda).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    row, dt = rnd(2, ch), rnd(2, h)
    cw, A, D = rnd(ch, w), -torch.rand(h, generator=g, device=cuda), rnd(h)
    c0, s0 = rnd(2, w - 1, ch), rnd(2, h, p, n)
    at = [slots - 1, 4097]
    conv, state = torch.zeros(slots, w - 1, ch, device=cuda), torch.zeros(slots, h, p, n, device=cuda)
    conv[at], state[at] = c0, s0
    out, want = torch.empty(2, inner, device=cuda), torch.empty(2, inner, device=cuda)
    k.ssm_token(out, row, dt, cw, None, conv, A, D, None, state, 2, h, p, gr, n, w,
                slots=torch.tensor(at, dtype=torch.int32, device=cuda))
    k.ssm_token(want, row, dt, cw, None, c0, A, D, None, s0, 2, h, p, gr, n, w)
    assert torch.equal(out, want) and torch.equal(conv[at], c0) and torch.equal(state[at], s0)
    state[at] = 0
    assert not state.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_of_empty_sequences_alone(k, cuda, dtype):
    """Tokens of no sequence, enough for the chunked form: nothing is written but zero states."""
    h, n, t = 4, 64, 200
    y = torch.full((t, h * 64), 9.0, dtype=dtype, device=cuda)
    v = torch.full((t, h * 64), float("nan"), dtype=dtype, device=cuda)
    state = torch.ones(3, h, 64, n, device=cuda)
    one = torch.ones(h, device=cuda)
    k.ssm_prompt(y, v, v[:, :h], -one, v[:, :n], v[:, :n], one, None, state,
                 torch.tensor([50, 50, 50, 50], dtype=torch.int32, device=cuda), 3, t, h, 64, 1, n,
                 has_state=torch.tensor([False, True, False], device=cuda))
    assert (y == 9).all() and (state[1] == 1).all() and not state[[0, 2]].any()
