"""The state-space operators against 64 bits, token by token.

Tolerances, per element, with `size` the same result of the absolute values of
every term (hybrid_ref): an f32 chain of n operations is off by at most
n * 2^-24 * size.  A term of the scan passes a product with exp(d A) per token
behind it (each off by at most 4 units: d, the product, exp, the multiply).
With bf16 activations an output's terms P[t][s] x[s] of its own chunk meet the
tensor cores with P rounded to bf16, off by at most half a step, 2^-8 of the
term, and the state before the chunk as two bf16 numbers, off by 2^-16: together
at most 2^-8 size.  States have no such term.  The output adds half a step of
its type."""

from __future__ import annotations

import pytest
import torch

import hybrid_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def k(cuda):
    from ervf_b200 import GPUKernels

    return GPUKernels()


def put(v, dev):
    return None if v is None else v.to(dev)


def ints(v, dev):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device=dev)


def packed(lens, lead=0):
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


# ------------------------------------------------------------- convolution

CONV = [  # lengths, tokens before the first sequence, behind the last
    ([1], 0, 0), ([5], 0, 0), ([33], 0, 2), ([100], 0, 0), ([0], 0, 0), ([0, 1, 2, 3, 4, 0], 3, 5),
    ([31, 32, 33, 0, 64, 1], 0, 0), ([2] * 40, 1, 1)]


@pytest.mark.parametrize("lens,lead,tail", CONV)
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_conv(k, cuda, lens, lead, tail, width, dtype):
    for channels in (1, 13, 64, 520):
        g = torch.Generator().manual_seed(channels)
        cu = packed(lens, lead)
        t, s = cu[-1] + tail, len(lens)
        x = torch.randn(t, channels, generator=g).to(dtype)
        w, b = torch.randn(channels, width, generator=g), torch.randn(channels, generator=g)
        state = torch.randn(s + 2, width - 1, channels, generator=g).to(dtype)
        slots = torch.randperm(s + 2, generator=g)[:s].tolist()
        has = [(i % 3) != 1 for i in range(s)]
        out = torch.full((t, channels), 9.0, dtype=dtype, device=cuda)
        st = state.to(cuda)
        k.conv1d_prompt(out, put(x, cuda), put(w, cuda), put(b, cuda), st, ints(cu, cuda), s, t, channels, width,
                        slots=ints(slots, cuda), has_state=torch.tensor(has, device=cuda))
        want, size, new = ref.conv(x, w, b, state, cu, slots, has)
        inside = slice(cu[0], cu[-1])
        ref.within(out[inside], want[inside], (ref.HALF[dtype] * want.abs() + 16 * ref.U * size)[inside] + 1e-30)
        assert (out[:lead] == 9).all() and (out[cu[-1]:] == 9).all()
        assert torch.equal(st.cpu().double(), new)


def test_conv_plain_call(k, cuda):
    """No state, no bias, no activation, one sequence, rows inside wider ones."""
    g = torch.Generator().manual_seed(0)
    wide = torch.randn(70, 100, generator=g).to(cuda)
    x, w = wide[:, 16:80], torch.randn(64, 4, generator=g)
    out = torch.empty(70, 64, device=cuda)
    k.conv1d_prompt(out, x, put(w, cuda), None, None, None, 1, 70, 64, 4, silu=False)
    want, size, _ = ref.conv(x.cpu(), w, None, None, [0, 70], None, None, use_silu=False)
    ref.within(out, want, ref.HALF[F32] * want.abs() + 16 * ref.U * size)


def test_conv_in_pieces_equals_whole(k, cuda):
    """A prompt fed in pieces through the carried state gives the bits of the whole."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(77, 48, generator=g).bfloat16().to(cuda), torch.randn(48, 4, generator=g).to(cuda)
    whole, state = torch.empty_like(x), torch.full((1, 3, 48), float("nan"), dtype=BF16, device=cuda)
    k.conv1d_prompt(whole, x, w, None, state, None, 1, 77, 48, 4)
    parts, st = torch.empty_like(x), torch.full((1, 3, 48), float("nan"), dtype=BF16, device=cuda)
    at = 0
    for n in (1, 2, 40, 0, 3, 31):
        k.conv1d_prompt(parts[at:at + n], x[at:at + n], w, None, st, None, 1, n, 48, 4,
                        has_state=torch.tensor([at > 0], device=cuda))
        at += n
    assert at == 77 and torch.equal(parts, whole) and torch.equal(st, state)


# -------------------------------------------------------------------- scan


def scan_case(lens, heads, head_dim, groups, d_state, dtype, lead=0, tail=0, seed=0, big_steps=False):
    g = torch.Generator().manual_seed(seed)
    cu = packed(lens, lead)
    t, s = cu[-1] + tail, len(lens)
    inner, bc = heads * head_dim, groups * d_state
    c = {"cu": cu, "t": t, "s": s, "dims": (heads, head_dim, groups, d_state)}
    c["xbc"] = torch.randn(t, inner + 2 * bc, generator=g).to(dtype)
    c["dt"] = torch.randn(t, heads, generator=g).to(dtype)
    c["A"] = -(1 + 15 * torch.rand(heads, generator=g))
    c["D"] = torch.randn(heads, generator=g)
    c["bias"] = torch.rand(heads, generator=g) * (2 if big_steps else 4) - (0 if big_steps else 6)
    c["state"] = torch.randn(s + 2, heads, head_dim, d_state, generator=g)
    c["slots"] = torch.randperm(s + 2, generator=g)[:s].tolist()
    c["has"] = [(i % 3) != 1 for i in range(s)]
    return c


def run_scan(k, cuda, c, dtype, slots=True, has=True, state=True, extras=True):
    h, p, gr, n = c["dims"]
    inner, bc = h * p, gr * n
    xbc, y = c["xbc"].to(cuda), torch.full((c["t"], inner), 9.0, dtype=dtype, device=cuda)
    st = c["state"].to(cuda, copy=True) if state else None
    k.ssm_prompt(y, xbc[:, :inner], put(c["dt"], cuda), put(c["A"], cuda), xbc[:, inner:inner + bc],
                 xbc[:, inner + bc:], put(c["D"], cuda) if extras else None, put(c["bias"], cuda) if extras else None,
                 st, ints(c["cu"], cuda), c["s"], c["t"], h, p, gr, n,
                 slots=ints(c["slots"], cuda) if slots else None,
                 has_state=torch.tensor(c["has"], device=cuda) if has else None)
    x, b, cc = c["xbc"].split([inner, bc, bc], 1)
    want = ref.scan(x.reshape(-1, h, p), c["dt"], c["A"], b.reshape(-1, gr, n), cc.reshape(-1, gr, n),
                    c["D"] if extras else None, c["bias"] if extras else None, c["state"] if state else None, c["cu"],
                    c["slots"] if slots else None, c["has"] if has else None)
    return y, st, want


def check_scan(y, st, want, c, dtype):
    ref_y, y_size, new, new_size = want
    chain = (4 * max(c["cu"][-1], 1) + 2 * c["dims"][3] + 32) * ref.U
    split = 2.0**-8 if dtype == BF16 else 0.0
    lo, hi = c["cu"][0], c["cu"][-1]
    flat, size = ref_y.flatten(1)[lo:hi], y_size.flatten(1)[lo:hi]
    ref.within(y[lo:hi], flat, ref.HALF[dtype] * (flat.abs() + split * size) + (split + chain) * size + 1e-30)
    assert (y[:lo] == 9).all() and (y[hi:] == 9).all()
    if st is not None:
        ref.within(st, new, ref.HALF[F32] * new.abs() + chain * new_size + 1e-30)


SCAN = [  # lengths, lead, tail
    ([1], 0, 0), ([0], 0, 1), ([15], 0, 0), ([64], 0, 0), ([127], 0, 3), ([128], 0, 0), ([129], 1, 0), ([300], 0, 0),
    ([0, 1, 130, 0, 63, 17, 0], 2, 3), ([5, 260, 128, 1], 0, 0)]


@pytest.mark.parametrize("lens,lead,tail", SCAN)
@pytest.mark.parametrize("d_state", [64, 128])
def test_scan_bf16(k, cuda, lens, lead, tail, d_state):
    c = scan_case(lens, 6, 64, 2, d_state, BF16, lead, tail)
    y, st, want = run_scan(k, cuda, c, BF16)
    check_scan(y, st, want, c, BF16)


@pytest.mark.parametrize("heads,head_dim,groups,d_state", [
    (1, 1, 1, 1), (3, 5, 3, 7), (4, 33, 1, 16), (2, 64, 2, 65), (2, 130, 1, 100), (2, 256, 1, 256), (5, 64, 1, 128)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_sizes(k, cuda, heads, head_dim, groups, d_state, dtype):
    c = scan_case([19, 0, 40], heads, head_dim, groups, d_state, dtype, 1, 2, seed=heads)
    y, st, want = run_scan(k, cuda, c, dtype)
    check_scan(y, st, want, c, dtype)


@pytest.mark.parametrize("lens,lead,tail", SCAN)
def test_scan_f32(k, cuda, lens, lead, tail):
    c = scan_case(lens, 4, 64, 2, 128, F32, lead, tail, seed=3)
    y, st, want = run_scan(k, cuda, c, F32)
    check_scan(y, st, want, c, F32)


@pytest.mark.parametrize("heads,groups", [(1, 1), (2, 2), (3, 1), (8, 1), (9, 1), (16, 2), (21, 3)])
def test_scan_heads_and_groups(k, cuda, heads, groups):
    c = scan_case([150, 20], heads, 64, groups, 128, BF16, seed=heads)
    y, st, want = run_scan(k, cuda, c, BF16)
    check_scan(y, st, want, c, BF16)


@pytest.mark.parametrize("lens,heads,groups,d_state", [
    ([2100], 64, 8, 128), ([700, 3, 0, 1290, 128, 64], 64, 8, 128), ([1500, 400], 40, 8, 64), ([3000], 16, 2, 128),
    ([257] * 9, 35, 7, 128)])
def test_scan_many_chunks(k, cuda, lens, heads, groups, d_state):
    """Several chunks to a CTA, pieces cut inside sequences and at their ends."""
    c = scan_case(lens, heads, 64, groups, d_state, BF16, 1, 2, seed=heads)
    for v in ("xbc", "dt", "A", "D", "bias", "state"):
        c[v] = c[v].to(cuda)  # the reference runs there too
    y, st, want = run_scan(k, cuda, c, BF16)
    check_scan(y, st, want, c, BF16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_large_steps(k, cuda, dtype):
    """Steps of several units: exp(d A) of a chunk underflows, nothing overflows."""
    c = scan_case([200, 140], 4, 64, 2, 128, dtype, seed=5, big_steps=True)
    c["dt"] *= 20
    y, st, want = run_scan(k, cuda, c, dtype)
    check_scan(y, st, want, c, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_steps_that_forget_everything(k, cuda, dtype):
    """A few steps of 30000 among ordinary ones: the exponents behind them keep their precision."""
    c = scan_case([200, 140], 4, 64, 2, 128, dtype, seed=8)
    c["dt"][7::40] = 30000.0
    y, st, want = run_scan(k, cuda, c, dtype)
    check_scan(y, st, want, c, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_no_decay(k, cuda, dtype):
    c = scan_case([200], 2, 64, 1, 128, dtype, seed=6)
    c["A"] *= 0
    y, st, want = run_scan(k, cuda, c, dtype)
    check_scan(y, st, want, c, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_defaults(k, cuda, dtype):
    """Without D, step bias, slots and flags every sequence starts from zero in its own slot; without
    a state nothing is kept."""
    c = scan_case([140, 3], 4, 64, 2, 128, dtype, seed=7)
    y, st, want = run_scan(k, cuda, c, dtype, slots=False, has=False, extras=False)
    check_scan(y, st, want, c, dtype)
    assert torch.equal(st[2:].cpu(), c["state"][2:])
    y2, _, _ = run_scan(k, cuda, c, dtype, slots=False, has=False, extras=False, state=False)
    assert torch.equal(y, y2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_slots_outside_the_state(k, cuda, dtype):
    c = scan_case([140, 30, 131], 4, 64, 2, 128, dtype, seed=8)
    c["slots"], c["has"] = [-1, 3, 99], [True, True, True]
    y, st, want = run_scan(k, cuda, c, dtype)
    check_scan(y, st, want, c, dtype)
    assert torch.equal(st[[0, 1, 2, 4]].cpu(), c["state"][[0, 1, 2, 4]])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_poison_stays_in_its_sequence(k, cuda, dtype):
    """NaN and infinities in a neighbour, in tokens of no sequence and in unused slots."""
    c = scan_case([100, 70, 150], 4, 64, 2, 128, dtype, 1, 2, seed=9)
    clean, st, want = run_scan(k, cuda, c, dtype)
    lo, hi = c["cu"][1], c["cu"][2]
    for name in ("xbc", "dt"):
        c[name][lo:hi] = float("nan")
        c[name][0] = c[name][-1] = float("inf")
    free = [i for i in range(5) if i not in c["slots"]]
    c["state"][free] = float("nan")
    c["state"][c["slots"][1]] = float("nan")
    y, st2, _ = run_scan(k, cuda, c, dtype)
    keep = list(range(1, lo)) + list(range(hi, c["cu"][3]))
    assert torch.equal(y[keep], clean[keep])
    for i in (0, 2):
        assert torch.equal(st2[c["slots"][i]], st[c["slots"][i]])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_in_pieces(k, cuda, dtype):
    """A prompt fed in pieces through the carried state stays within the whole's tolerance."""
    c = scan_case([290], 4, 64, 2, 128, dtype, seed=10)
    c["slots"], c["has"], cuts = [1], [True], [0, 130, 131, 140, 290]
    h, p, gr, n = c["dims"]
    inner, bc = h * p, gr * n
    want = run_scan(k, cuda, c, dtype)[2]
    xbc, dt, y = c["xbc"].to(cuda), c["dt"].to(cuda), torch.empty(290, inner, dtype=dtype, device=cuda)
    st = c["state"].to(cuda)
    for a, b in zip(cuts, cuts[1:]):
        k.ssm_prompt(y[a:b], xbc[a:b, :inner], dt[a:b], put(c["A"], cuda), xbc[a:b, inner:inner + bc],
                     xbc[a:b, inner + bc:], put(c["D"], cuda), put(c["bias"], cuda), st, None, 1, b - a, h, p, gr, n,
                     slots=ints([1], cuda), has_state=torch.tensor([True], device=cuda))
    check_scan(y, st, want, c, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_same_bits_two_streams_and_graph(k, cuda, dtype):
    """Two calls at once on two streams and a replayed graph give the first call's bits."""
    from ervf_b200 import GPUKernels

    c = scan_case([500, 77], 8, 64, 2, 128, dtype, seed=11)
    h, p, gr, n = c["dims"]
    inner, bc = h * p, gr * n
    xbc, dt, A, D, bias = (put(c[v], cuda) for v in ("xbc", "dt", "A", "D", "bias"))
    cu, slots, has = ints(c["cu"], cuda), ints(c["slots"], cuda), torch.tensor(c["has"], device=cuda)

    def call(kern, y, st):
        kern.ssm_prompt(y, xbc[:, :inner], dt, A, xbc[:, inner:inner + bc], xbc[:, inner + bc:], D, bias, st, cu, 2,
                        577, h, p, gr, n, slots=slots, has_state=has)

    ys = [torch.zeros(577, inner, dtype=dtype, device=cuda) for _ in range(4)]
    sts = [c["state"].to(cuda) for _ in range(4)]
    call(k, ys[0], sts[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    kernels = [GPUKernels() for _ in range(2)]
    for i in range(2):
        kernels[i].stream = streams[i]
        call(kernels[i], ys[1 + i], sts[1 + i])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(k, ys[3], sts[3])
    sts[3].copy_(c["state"])
    g.replay()
    torch.cuda.synchronize()
    for i in (1, 2, 3):
        assert torch.equal(ys[i], ys[0]) and torch.equal(sts[i], sts[0])


# --------------------------------------------------------------- one token


def token_case(seqs, heads, head_dim, groups, d_state, width, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    inner = heads * head_dim
    ch = inner + 2 * groups * d_state
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"row": rnd(seqs, inner + ch + heads + 3).to(dtype), "cw": rnd(ch, width) * 0.5, "cb": rnd(ch) * 0.1,
            "conv": rnd(seqs + 2, width - 1, ch).to(dtype), "A": -(1 + 15 * torch.rand(heads, generator=g)),
            "D": rnd(heads), "bias": torch.rand(heads, generator=g) * 4 - 6,
            "state": rnd(seqs + 2, heads, head_dim, d_state), "nw": rnd(inner),
            "slots": torch.randperm(seqs + 2, generator=g)[:seqs].tolist(),
            "dims": (heads, head_dim, groups, d_state), "s": seqs, "w": width}


def run_token(k, cuda, c, dtype, z=True, norm=True, extras=True):
    h, p, gr, n = c["dims"]
    inner = h * p
    ch = inner + 2 * gr * n
    row, conv, state = c["row"].to(cuda), c["conv"].to(cuda), c["state"].to(cuda)
    out = torch.full((c["s"], inner), 9.0, dtype=dtype, device=cuda)
    k.ssm_token(out, row[:, inner:inner + ch], row[:, inner + ch:], put(c["cw"], cuda),
                put(c["cb"], cuda) if extras else None, conv, put(c["A"], cuda), put(c["D"], cuda) if extras else None,
                put(c["bias"], cuda) if extras else None, state, c["s"], h, p, gr, n, c["w"],
                z=row[:, :inner] if z else None, norm_w=put(c["nw"], cuda) if norm else None,
                slots=ints(c["slots"], cuda))
    return out, conv, state


def check_token(c, dtype, got, z=True, norm=True, extras=True):
    out, conv, state = got
    h, p, gr, n = c["dims"]
    inner, s = h * p, c["s"]
    ch = inner + 2 * gr * n
    cu = list(range(s + 1))
    has = [True] * s
    v, v_size, new_conv = ref.conv(c["row"][:, inner:inner + ch], c["cw"], c["cb"] if extras else None, c["conv"], cu,
                                   c["slots"], has)
    assert torch.equal(conv.cpu().double(), new_conv)
    x, b, cc = v.split([inner, gr * n, gr * n], 1)
    dt = c["row"][:, inner + ch:inner + ch + h]
    y, y_size, new, new_size = ref.scan(x.reshape(s, h, p), dt, c["A"], b.reshape(s, gr, n), cc.reshape(s, gr, n),
                                        c["D"] if extras else None, c["bias"] if extras else None, c["state"], cu,
                                        c["slots"], has)
    # the convolution's outputs are off by 16 units of their size; x, B and C
    # carry that into every product of two of them
    amp = float((v_size / v.abs().clamp(min=1e-3)).max()) * 16
    chain = (64 + 2 * n) * ref.U
    vs = [t.reshape(s, -1, t.shape[1] // q) for t, q in zip(v_size.split([inner, gr * n, gr * n], 1), (h, gr, gr))]
    grow = ref.scan(vs[0], dt, c["A"], vs[1], vs[2], c["D"].abs() if extras else None, c["bias"] if extras else None,
                    c["state"].abs(), cu, c["slots"], has)
    assert amp > 0
    ref.within(state, new, ref.HALF[F32] * new.abs() + (chain + 48 * ref.U) * grow[2].abs() + 1e-30)
    y, err = y.flatten(1), (chain + 64 * ref.U) * grow[1].flatten(1)
    if z:
        gate = ref.silu(c["row"][:, :inner].double())
        y, err = y * gate, err * gate.abs() + 8 * ref.U * (y * gate).abs()
    if norm:
        gy = y.reshape(s, gr, -1)
        rms = torch.sqrt(gy.square().mean(-1, keepdim=True) + 1e-5)
        e = err.reshape(s, gr, -1)
        # the mean's own error: first order in the errors, and a chain of its terms
        worst = torch.sqrt(e.square().mean(-1, keepdim=True)) / rms
        err = ((e / rms) + (gy / rms).abs() * (worst + (p * h // gr + 16) * ref.U)).reshape(s, -1) * c["nw"].abs()
        y = (gy / rms).reshape(s, -1) * c["nw"].double()
    ref.within(out, y, ref.HALF[dtype] * (y.abs() + err) + err + 1e-30)


@pytest.mark.parametrize("seqs,heads,head_dim,groups,d_state,width", [
    (1, 1, 1, 1, 4, 2), (1, 8, 64, 1, 128, 4), (3, 6, 64, 2, 128, 4), (5, 9, 33, 1, 64, 3), (2, 16, 64, 2, 96, 4),
    (4, 11, 64, 1, 128, 4), (2, 20, 32, 1, 256, 4), (7, 3, 256, 3, 16, 2), (33, 8, 64, 8, 128, 4), (230, 64, 256, 1, 4, 2), (200, 16, 64, 8, 128, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_token(k, cuda, seqs, heads, head_dim, groups, d_state, width, dtype):
    c = token_case(seqs, heads, head_dim, groups, d_state, width, dtype, seed=seqs)
    check_token(c, dtype, run_token(k, cuda, c, dtype))


@pytest.mark.parametrize("z,norm,extras", [(False, True, True), (True, False, True), (False, False, False)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_token_parts(k, cuda, z, norm, extras, dtype):
    c = token_case(3, 6, 64, 2, 128, 4, dtype, seed=4)
    check_token(c, dtype, run_token(k, cuda, c, dtype, z, norm, extras), z, norm, extras)


def test_token_padded_rows(k, cuda):
    """Rows of a padded batch name no slot: they start from zero and store nothing."""
    c = token_case(4, 6, 64, 2, 128, 4, F32, seed=5)
    c["slots"] = [2, -1, 5, 77]
    got = run_token(k, cuda, c, F32)
    check_token(c, F32, got)
    assert torch.equal(got[2][[0, 1, 3, 4]].cpu(), c["state"][[0, 1, 3, 4]])
    assert torch.equal(got[1][[0, 1, 3, 4]].cpu(), c["conv"][[0, 1, 3, 4]])


def test_token_captured_and_replayed(k, cuda):
    c = token_case(2, 8, 64, 2, 128, 4, BF16, seed=6)
    h, p, gr, n = c["dims"]
    inner, ch = h * p, h * p + 2 * gr * n
    dev = {v: c[v].to(cuda) for v in ("row", "conv", "state", "cw", "cb", "A", "D", "bias", "nw")}
    slots, out = ints(c["slots"], cuda), torch.zeros(2, inner, dtype=BF16, device=cuda)

    def call():
        k.ssm_token(out, dev["row"][:, inner:inner + ch], dev["row"][:, inner + ch:], dev["cw"], dev["cb"],
                    dev["conv"], dev["A"], dev["D"], dev["bias"], dev["state"], 2, h, p, gr, n, 4,
                    z=dev["row"][:, :inner], norm_w=dev["nw"], slots=slots)

    want = []
    for _ in range(3):
        call()
        want.append((out.clone(), dev["conv"].clone(), dev["state"].clone()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    dev["conv"].copy_(c["conv"])
    dev["state"].copy_(c["state"])
    for o, cv, st in want:
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(dev["conv"], cv) and torch.equal(dev["state"], st)


# -------------------------------------------------------------- gated norm


@pytest.mark.parametrize("tokens,groups,size", [
    (1, 1, 1), (3, 2, 7), (5, 8, 512), (40, 1, 64), (2, 3, 1000), (3, 1, 4096), (2, 1, 10000), (200, 4, 72)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gate", [True, False])
def test_gated_norm(k, cuda, tokens, groups, size, dtype, gate):
    g = torch.Generator().manual_seed(size)
    n = groups * size
    y, z = (torch.randn(tokens, n, generator=g).to(dtype) for _ in range(2))
    w = torch.randn(n, generator=g)
    y[0] = 0  # a group of zeros
    out = torch.empty(tokens, n, dtype=dtype, device=cuda)
    k.gated_norm(out, put(y, cuda), put(z, cuda) if gate else None, put(w, cuda), tokens, groups, size)
    want, s = ref.gated_norm(y, z if gate else None, w, groups, 1e-5)
    b = ref.HALF[dtype] * want.abs() + (size / 2 + 32) * ref.U * s + 1e-30
    ref.within(out, want, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_norm_in_place_and_strided(k, cuda, dtype):
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(30, 700, generator=g).to(dtype)
    dev = wide.to(cuda)
    w = torch.randn(256, generator=g)
    y, z = dev[:, 3:259], dev[:, 300:556]
    k.gated_norm(y, y, z, put(w, cuda), 30, 2, 128)
    want, s = ref.gated_norm(wide[:, 3:259], wide[:, 300:556], w, 2, 1e-5)
    ref.within(y, want, ref.HALF[dtype] * want.abs() + 96 * ref.U * s + 1e-30)
    assert torch.equal(dev[:, 259:].cpu(), wide[:, 259:]) and torch.equal(dev[:, :3].cpu(), wide[:, :3])


# ---------------------------------------------------------- a layer's chain


@pytest.mark.parametrize("lens", [[70], [1, 140, 6]])
def test_prompt_then_tokens_through_a_layer(k, cuda, lens):
    """Projection, convolution, scan, norm, projection onto the residual for a prompt, then two
    decoded tokens of each sequence through the one-token step: against the same chain in 64 bits on the
    values that each operator was given (bf16 between them)."""
    hidden, heads, p, gr, n, width = 128, 4, 64, 2, 64, 4
    inner, ch = heads * p, heads * p + 2 * gr * n
    rows = inner + ch + 8  # 8 step columns: 4 used
    g = torch.Generator().manual_seed(len(lens))
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    win, wout = (rnd(rows, hidden) * 0.08).bfloat16(), (rnd(hidden, inner) * 0.06).bfloat16()
    cw, cb, nw = rnd(ch, width) * 0.5, rnd(ch) * 0.1, rnd(inner)
    A, D, bias = -(1 + 3 * torch.rand(heads, generator=g)), rnd(heads), rnd(heads) * 0.5 - 2
    cu, s = packed(lens), len(lens)
    t = cu[-1]
    par = [put(v, cuda) for v in (win, wout, cw, cb, nw, A, D, bias)]
    conv = torch.zeros(s, width - 1, ch, dtype=BF16, device=cuda)
    state = torch.zeros(s, heads, p, n, device=cuda)

    def project(W, x, out, resid=None):
        k.linear_bf16(out, W, x, out.shape[1], x.shape[1], x.shape[0], resid=resid)
        want, size = ref.linear(W.cpu(), x.cpu(), None, "none", None if resid is None else resid.cpu())
        ref.within(out, want, ref.HALF[out.dtype] * want.abs() + (2 * x.shape[1] + 32) * ref.U * size + 1e-30)
        return out

    h = rnd(t, hidden).bfloat16().to(cuda)
    zx = project(par[0], h, torch.empty(t, rows, dtype=BF16, device=cuda))
    xbc = torch.empty(t, ch, dtype=BF16, device=cuda)
    k.conv1d_prompt(xbc, zx[:, inner:inner + ch], par[2], par[3], conv, ints(cu, cuda), s, t, ch, width)
    want, size, ref_conv = ref.conv(zx[:, inner:inner + ch].cpu(), cw, cb, torch.zeros(s, width - 1, ch), cu, None, None)
    ref.within(xbc, want, ref.HALF[BF16] * want.abs() + 16 * ref.U * size + 1e-30)
    assert torch.equal(conv.cpu().double(), ref_conv)
    y = torch.empty(t, inner, dtype=BF16, device=cuda)
    dt = zx[:, inner + ch:inner + ch + heads]
    k.ssm_prompt(y, xbc[:, :inner], dt, par[5], xbc[:, inner:inner + gr * n], xbc[:, inner + gr * n:], par[6], par[7],
                 state, ints(cu, cuda), s, t, heads, p, gr, n)
    x, b, c = xbc.cpu().split([inner, gr * n, gr * n], 1)
    want = ref.scan(x.reshape(t, heads, p), dt.cpu(), A, b.reshape(t, gr, n), c.reshape(t, gr, n), D, bias,
                    torch.zeros(s, heads, p, n), cu, None, None)
    case = {"cu": cu, "dims": (heads, p, gr, n)}
    check_scan(y, state, want, case, BF16)
    ng = torch.empty_like(y)
    k.gated_norm(ng, y, zx[:, :inner], par[4], t, gr, inner // gr)
    want, size = ref.gated_norm(y.cpu(), zx[:, :inner].cpu(), nw, gr, 1e-5)
    ref.within(ng, want, ref.HALF[BF16] * want.abs() + (inner // gr / 2 + 32) * ref.U * size + 1e-30)
    stream = rnd(t, hidden).to(cuda)
    project(par[1], ng, torch.empty(t, hidden, device=cuda), resid=stream)

    for step in range(2):
        h1 = rnd(s, hidden).bfloat16().to(cuda)
        row = project(par[0], h1, torch.empty(s, rows, dtype=BF16, device=cuda))
        c = {"row": row[:, :inner + ch + heads].cpu(), "cw": cw, "cb": cb, "conv": conv.cpu(), "A": A, "D": D,
             "bias": bias, "state": state.cpu(), "nw": nw, "slots": list(range(s)), "dims": (heads, p, gr, n), "s": s,
             "w": width}
        out = torch.empty(s, inner, dtype=BF16, device=cuda)
        k.ssm_token(out, row[:, inner:inner + ch], row[:, inner + ch:], par[2], par[3], conv, par[5], par[6], par[7],
                    state, s, heads, p, gr, n, width, z=row[:, :inner], norm_w=par[4])
        check_token(c, BF16, (out, conv, state))
        project(par[1], out, torch.empty(s, hidden, device=cuda), resid=rnd(s, hidden).to(cuda))
