"""Infinities and NaN in the scan's inputs: they reach what the recurrence lets
them reach, and nothing else."""

from __future__ import annotations

import pytest
import torch

import hybrid_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


@pytest.fixture(scope="module")
def k(cuda):
    from ervf_b200 import GPUKernels

    return GPUKernels()


@pytest.mark.parametrize("d_state", [1, 5, 16, 40, 64, 100, 130])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_infinity_with_any_number_of_states(k, cuda, d_state, dtype):
    """All terms positive: the output of an infinite input, and of the tokens behind it, is infinite
    and no NaN, however many columns the kernel pads the state with."""
    g = torch.Generator().manual_seed(d_state)
    t, p = 20, 3
    x, b, c = (torch.rand(t, w, generator=g).to(dtype) + 0.5 for w in (p, d_state, d_state))
    x[7, 1] = INF
    y, state = torch.zeros(t, p, dtype=dtype, device=cuda), torch.zeros(1, 1, p, d_state, device=cuda)
    one = torch.ones(1, device=cuda)
    k.ssm_prompt(y, x.to(cuda), torch.zeros(t, 1, dtype=dtype, device=cuda), -one, b.to(cuda), c.to(cuda), one, None,
                 state, None, 1, t, 1, p, 1, d_state)
    want = torch.zeros(t, p, dtype=torch.bool)
    want[7:, 1] = True
    y = y.float().cpu()
    assert torch.equal(y == INF, want) and not torch.isnan(y).any()
    assert (state[0, 0, 1] == INF).all() and torch.isfinite(state[0, 0, [0, 2]]).all()


@pytest.mark.parametrize("d_state", [4, 28, 32, 48, 64, 100, 132, 256])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_token_infinity_with_any_number_of_states(k, cuda, d_state, dtype):
    p = 3
    ch = p + 2 * d_state
    row = torch.ones(1, ch, dtype=dtype, device=cuda)
    row[0, 1] = INF
    cw = torch.zeros(ch, 2, device=cuda)
    cw[:, 1] = 1
    one = torch.ones(1, device=cuda)
    out = torch.zeros(1, p, dtype=dtype, device=cuda)
    conv, state = torch.zeros(1, 1, ch, dtype=dtype, device=cuda), torch.ones(1, 1, p, d_state, device=cuda)
    k.ssm_token(out, row, torch.zeros(1, 1, dtype=dtype, device=cuda), cw, None, conv, -one, one, None, state, 1, 1, p, 1,
                d_state, 2)
    assert (out[0].float().cpu() == INF).tolist() == [False, True, False] and not torch.isnan(out).any()
    assert (state[0, 0, 1] == INF).all() and torch.isfinite(state[0, 0, [0, 2]]).all()


def poisoned(what, value, dtype, d_state):
    """A pack with `value` in a few places of one input, and which outputs [token, head, p] and
    states [slot, head, p, n] the recurrence lets these reach."""
    from test_ssm_gpu import scan_case

    h, p, gr = 6, 64, 2
    c = scan_case([200, 90, 0, 133, 1], h, p, gr, d_state, dtype, 1, 2, seed=d_state)
    inner, bc, per = h * p, gr * d_state, h // gr
    cu = c["cu"]
    reach = torch.zeros(c["t"], h, p, dtype=torch.bool)
    kept = torch.zeros_like(c["state"], dtype=torch.bool)
    clean = {v: c[v].clone() for v in ("xbc", "dt")}
    # the first and last token of a sequence, and of chunks and blocks of 32 inside them
    for i, t in enumerate((cu[0] + 127, cu[0] + 130, cu[1] + 31, cu[2] - 1, cu[3] + 64, cu[3] + 100, cu[4])):
        seq = max(s for s in range(c["s"]) if cu[s] <= t < cu[s + 1])
        tokens, slot = slice(t, cu[seq + 1]), c["slots"][seq]
        head, col, n = (i * 5) % h, (i * 29 + 3) % p, (i * 37 + 2) % d_state
        g = head // per
        heads = slice(g * per, (g + 1) * per)
        if what == "x":
            c["xbc"][t, head * p + col] = value
            reach[tokens, head, col] = True
            kept[slot, head, col] = True
        elif what == "B":
            c["xbc"][t, inner + g * d_state + n] = value
            reach[tokens, heads] = True
            kept[slot, heads, :, n] = True
        elif what == "C":
            c["xbc"][t, inner + bc + g * d_state + n] = value
            reach[t, heads] = True
        else:
            c["dt"][t, head] = value
            reach[tokens, head] = True
            kept[slot, head] = True
    return c, clean, reach, kept


@pytest.mark.parametrize("what,value", [("x", float("nan")), ("x", INF), ("x", -INF), ("B", float("nan")),
                                        ("B", INF), ("C", float("nan")), ("C", INF), ("dt", float("nan"))])
@pytest.mark.parametrize("dtype,d_state", [(F32, 64), (BF16, 64), (BF16, 128)])
def test_scan_poison_reaches_no_token_before_it(k, cuda, what, value, dtype, d_state):
    """Everything it does not reach is what it is without it, within the same tolerance; everything it
    does is not finite."""
    from test_ssm_gpu import run_scan

    c, clean, reach, kept = poisoned(what, value, dtype, d_state)
    y, st, _ = run_scan(k, cuda, c, dtype)
    c.update(clean)
    _, _, (ref_y, y_size, new, new_size) = run_scan(k, cuda, c, dtype)
    lo, hi = c["cu"][0], c["cu"][-1]
    y, st = y.double().cpu().view(reach.shape)[lo:hi], st.double().cpu()
    assert not torch.isfinite(y[reach[lo:hi]]).any() and not torch.isfinite(st[kept]).any()
    chain = (4 * hi + 2 * d_state + 32) * ref.U
    split = 2.0**-8 if dtype == BF16 else 0.0
    want, size = ref_y[lo:hi], y_size[lo:hi]
    bound = ref.HALF[dtype] * (want.abs() + split * size) + (split + chain) * size + 1e-30
    ok = ~reach[lo:hi]
    ref.within(y[ok], want[ok], bound[ok])
    ref.within(st[~kept], new[~kept], (ref.HALF[F32] * new.abs() + chain * new_size + 1e-30)[~kept])
