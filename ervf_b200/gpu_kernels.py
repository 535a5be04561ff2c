"""``GPUKernels`` -- the dense and state-space half of the reference's kernel
wrapper (kennydd001/ervf src/moe_lab/lightningstream_nemotron/gpu_kernels.py)
on the B200 C ABI:

  * ``mv_bf16`` / ``mv_f32`` (:1549-1555), the BF16 dense GEMV and the FP32
    router GEMV, plus batched BF16 forms;
  * ``linear_bf16``, the dense projection of any number of tokens with bias,
    activation and residual in its epilogue;
  * ``conv1d_prompt``, ``ssm_prompt``, ``gated_norm``: the hybrid's state-space
    layers for packed prompts, and ``ssm_token`` for one token of each
    sequence (the reference's conv1d, softplus, ssm and gated_rmsnorm,
    :77-1515, run one token of one sequence).

The reference's attention kernels are out of scope.

Buffers of the projection and state-space methods are caller-owned CUDA
tensors on this object's device, activations in one row per token.  A 2-D
tensor may have any row stride (a slice of a wider row); other shapes are
read as contiguous rows.  Objects with ``__cuda_array_interface__`` and int
addresses are contiguous rows too, and an int output needs ``dtype``.

Launches go on ``self.stream`` if set (a torch or CuPy stream or a raw handle),
else on torch's current stream -- with CuPy too: a program whose arrays are on
a CuPy stream sets it.
"""

from __future__ import annotations

import torch

from . import _lib
from .fused_nvfp4 import _need, current_stream, ptr

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.uint16: _lib.BF16,
          torch.int16: _lib.BF16}
_CAI_TYPES = {"<f4": _lib.F32, "<u2": _lib.BF16, "<i2": _lib.BF16}
_ACTS = {"none": _lib.ACT_NONE, "relu2": _lib.ACT_RELU2, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
_F32, _I32, _U8 = (torch.float32,), (torch.int32,), (torch.uint8, torch.bool)
_BF16 = (torch.bfloat16, torch.uint16, torch.int16)
_CODE_TYPES = {_lib.F32: _F32, _lib.BF16: _BF16}
_CAI_NAMES = {_F32: ("<f4",), _I32: ("<i4",), _U8: ("|u1", "|b1"), _BF16: ("<u2", "<i2")}


# handle of torch's current stream on a device, without making a Stream object
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: int(torch.cuda.current_stream(index).cuda_stream))


def _type_of(a, dtype, what: str) -> int:
    """Element type code of an activation array (f32, or bf16 as such or as its bits)."""
    if isinstance(a, torch.Tensor):
        code = _TYPES.get(a.dtype)
    elif isinstance(a, int):
        code = _TYPES.get(dtype)
    else:
        code = _CAI_TYPES.get(a.__cuda_array_interface__["typestr"])
    if code is None:
        raise ValueError(f"{what}: float32 or bfloat16 elements are needed")
    return code


def _fit(*sizes) -> None:
    """Sizes reach the C ABI as 32-bit numbers, to which ctypes would cut them without a word.
    Called where one of them has a bit above the 31st (or a sign, which the C ABI refuses)."""
    if max(sizes) > 0x7FFFFFFF or min(sizes) < -0x80000000:
        raise ValueError(f"unsupported shape: sizes {sizes} pass 32 bits")


def _contiguous(cai) -> bool:
    """Whether a CUDA array's elements lie in C order without gaps."""
    strides, step = cai.get("strides"), int(cai["typestr"][2:])
    if strides is None:
        return True
    for n, s in zip(reversed(cai["shape"]), reversed(strides)):
        if n > 1 and s != step:
            return False
        step *= n
    return True


class GPUKernels:
    def __init__(self, block: int = 256, device=None):
        _lib.load()
        self.block = block
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None \
            else torch.device(device)
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._index = self.device.index
        self.stream = None

    def _s(self) -> int:
        if self.stream is not None:
            return current_stream(self.stream, self.device)
        return int(torch.cuda.current_stream(self.device).cuda_stream)

    def mv_bf16(self, out, W, x, rows: int, cols: int) -> None:
        """out[rows] = bf16 W[rows, cols] @ x[cols] (fp32), bit-exact to the
        reference's gemv_bf16."""
        self.mv_bf16_batched(out, W, x, rows, cols, 1)

    def mm_bf16_tc(self, out, W, x, rows: int, cols: int, batch: int) -> None:
        """out[b*rows + r] for x[b*cols + k], b < batch <= 8, on the tensor
        cores (tolerance path: rel-L2 <= 1e-3, not gemv_bf16's chain order)."""
        _need(out, batch * rows, "out")
        _need(W, rows * cols, "W")
        _need(x, batch * cols, "x")
        _lib.call("ervf_bf16_gemm_tc", ptr(W), ptr(x), ptr(out), int(rows), int(cols), int(batch),
                  self._s())

    def mv_bf16_batched(self, out, W, x, rows: int, cols: int, batch: int) -> None:
        """out[b*rows + r] for x[b*cols + k], b < batch <= 8."""
        _need(out, batch * rows, "out")
        _need(W, rows * cols, "W")
        _need(x, batch * cols, "x")
        _lib.call("ervf_bf16_gemv", ptr(W), ptr(x), ptr(out), int(rows), int(cols), int(batch),
                  self._s())

    def mv_f32(self, out, W, x, rows: int, cols: int) -> None:
        """out[rows] = fp32 W[rows, cols] @ x[cols], bit-exact to the
        reference's gemv_f32 (the router projection, gpu_kernels.py:51-74)."""
        _need(out, rows, "out")
        _need(W, rows * cols, "W")
        _need(x, cols, "x")
        _lib.call("ervf_f32_gemv", ptr(W), ptr(x), ptr(out), int(rows), int(cols), self._s())

    # ------------------------------------------------ argument checks
    # A call's checks are part of a decode step's latency: the accepted case
    # is decided with few attribute reads, the error text made afterwards.
    def _rows(self, a, rows: int, cols: int, code, what: str) -> tuple[int, int]:
        """Address and row stride of an activation array of `rows` rows."""
        if a is None:
            return 0, cols
        if isinstance(a, torch.Tensor):
            if a.get_device() == self._index and _TYPES.get(a.dtype) == code:
                if a.dim() == 2:
                    r, c = a.shape
                    stride = a.stride()
                    if r >= rows and c >= cols and (stride[1] == 1 or cols == 1):
                        return a.data_ptr(), stride[0] if rows > 1 else cols
                if a.numel() >= rows * cols and a.is_contiguous():
                    return a.data_ptr(), cols
            self._refuse(a, rows * cols, _CODE_TYPES[code], what)
        if not isinstance(a, int):
            if _type_of(a, None, what) != code:
                raise ValueError(f"{what}: its elements do not fit the other arrays")
            if not _contiguous(a.__cuda_array_interface__):
                raise ValueError(f"{what}: a contiguous array is needed")
            _need(a, rows * cols, what)
        return ptr(a), cols

    def _flat(self, a, n: int, dtypes, what: str) -> int:
        """Address of a contiguous parameter, state or index array (None: 0)."""
        if a is None:
            return 0
        if isinstance(a, torch.Tensor):
            if (a.get_device() == self._index and a.dtype in dtypes and a.numel() >= n
                    and a.is_contiguous()):
                return a.data_ptr()
            self._refuse(a, n, dtypes, what)
        if not isinstance(a, int):
            cai = a.__cuda_array_interface__
            if cai["typestr"] not in _CAI_NAMES[dtypes] or not _contiguous(cai):
                raise ValueError(f"{what}: a contiguous array of {_CAI_NAMES[dtypes]} is needed, not "
                                 f"{cai['typestr']} with strides {cai.get('strides')}")
            _need(a, n, what)
        return ptr(a)

    def _refuse(self, a, n: int, dtypes, what: str):
        if a.get_device() != self._index:
            raise ValueError(f"{what} is on {a.device}, this object launches on {self.device}")
        if a.dtype not in dtypes:
            raise ValueError(f"{what}: elements of type {a.dtype} do not fit, one of {dtypes} is needed")
        if a.numel() < n:
            raise ValueError(f"{what} holds {a.numel()} elements, needs {n}")
        raise ValueError(f"{what}: rows of contiguous elements, {n} in all, are needed")

    @staticmethod
    def _slots_of(state, per_slot: int, n_slots, what: str) -> int:
        if n_slots is not None:
            _fit(int(n_slots))
            return int(n_slots)
        if state is None:
            return 0
        if not isinstance(state, torch.Tensor):
            raise ValueError(f"{what}: n_slots is needed beside an address")
        return min(state.numel() // max(per_slot, 1), 0x7FFFFFFF)  # slots are named by 32-bit numbers

    def _launch(self, name: str, *args) -> None:
        stream = _raw_stream(self._index) if self.stream is None else current_stream(self.stream, self.device)
        if torch.cuda.current_device() == self._index:
            _lib.call(name, *args, stream)
        else:
            with torch.cuda.device(self.device):
                _lib.call(name, *args, stream)

    # ------------------------------------------------ dense projection
    def linear_bf16(self, out, W, x, rows: int, cols: int, tokens: int, bias=None, act: str = "none",
                    resid=None, dtype=None) -> None:
        """out[t] = act(bf16 W[rows, cols] @ bf16 x[t] + bias) + resid[t] for any number of tokens.
        out (f32 or bf16) and resid have one type; bias is f32; act is "none",
        "relu2", "silu" or "gelu"; resid may be out itself.  f32 sums and
        epilogue, one rounding, the same bits on every call."""
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}, got {act!r}")
        if (rows | cols | tokens) >> 31:
            _fit(rows, cols, tokens)
        code = _type_of(out, dtype, "out")
        po, so = self._rows(out, tokens, rows, code, "out")
        px, sx = self._rows(x, tokens, cols, _lib.BF16, "x")
        pr, sr = self._rows(resid, tokens, rows, code, "resid")
        pw = self._flat(W, rows * cols, _BF16, "W")
        pb = self._flat(bias, rows, _F32, "bias")
        self._launch("ervf_linear_bf16", pw, px, sx, pb, pr, sr, po, so, code, rows, cols, tokens, _ACTS[act])

    # ------------------------------------------------ state-space layers
    def conv1d_prompt(self, out, x, w, bias, state, cu_seqlens, seqs: int, tokens: int, channels: int,
                      width: int, slots=None, has_state=None, silu: bool = True, n_slots=None,
                      dtype=None) -> None:
        """Causal depthwise convolution of packed prompts, out[t][c] = silu(bias[c] +
        sum_j w[c][j] x[t - width + 1 + j][c]).  Sequence i is tokens
        cu_seqlens[i] .. cu_seqlens[i + 1] (int32 on the device; None: one
        sequence of all tokens).  state [n_slots, width - 1, channels] (None: no
        sequence carries any): row slots[i] (None: i) holds the inputs before
        sequence i where has_state[i], and its last inputs afterwards; a slot
        outside the array is no state.  No slot may be named twice."""
        if (seqs | tokens | channels | width) >> 31:
            _fit(seqs, tokens, channels, width)
        code = _type_of(out, dtype, "out")
        po, so = self._rows(out, tokens, channels, code, "out")
        px, sx = self._rows(x, tokens, channels, code, "x")
        ns = self._slots_of(state, (width - 1) * channels, n_slots, "state")
        self._launch("ervf_conv1d_prompt", px, sx, self._flat(w, channels * width, _F32, "w"),
                     self._flat(bias, channels, _F32, "bias"),
                     self._flat(state, ns * (width - 1) * channels, _CODE_TYPES[code], "state"), ns,
                     self._flat(slots, seqs, _I32, "slots"), self._flat(has_state, seqs, _U8, "has_state"),
                     self._flat(cu_seqlens, seqs + 1, _I32, "cu_seqlens"), seqs, po, so, code, tokens,
                     channels, width, 1 if silu else 0)

    def ssm_prompt(self, y, x, dt, A, B, C, D, dt_bias, state, cu_seqlens, seqs: int, tokens: int,
                   heads: int, head_dim: int, groups: int, d_state: int, slots=None, has_state=None,
                   n_slots=None, dtype=None) -> None:
        """Selective scan of packed prompts: with d_t = softplus(dt[t][h] + dt_bias[h]),
        S_t = exp(d_t A[h]) S_{t-1} + d_t x[t][h] B[t][g]^T and y[t][h] = S_t C[t][g] +
        D[h] x[t][h].  state f32 [n_slots, heads, head_dim, d_state] or None;
        cu_seqlens, slots and has_state as in conv1d_prompt.  A is not above 0.
        bf16 with head_dim 64, d_state 64 or 128, rows of x, B, C and y of 16-byte
        alignment, more than 32 tokens and at most 16384 sequences runs in chunks on
        the tensor cores, where the weights of a chunk's tokens are rounded to bf16
        (y is off by a tenth more than its own rounding; states stay f32);
        everything else token by token in f32, a long prompt in 25 to 30 times the
        time."""
        if (seqs | tokens | heads | head_dim | groups | d_state) >> 31:
            _fit(seqs, tokens, heads, head_dim, groups, d_state)
        code = _type_of(y, dtype, "y")
        inner, bc = heads * head_dim, groups * d_state
        py, sy = self._rows(y, tokens, inner, code, "y")
        px, sx = self._rows(x, tokens, inner, code, "x")
        pd, sd = self._rows(dt, tokens, heads, code, "dt")
        pb, sb = self._rows(B, tokens, bc, code, "B")
        pc, sc = self._rows(C, tokens, bc, code, "C")
        ns = self._slots_of(state, inner * d_state, n_slots, "state")
        nb = _lib.load().ervf_ssm_prompt_scratch_bytes(code, tokens, seqs, heads, head_dim, groups, d_state)
        scratch = self._scratch(nb)
        self._launch("ervf_ssm_prompt", px, sx, pd, sd, self._flat(A, heads, _F32, "A"), pb, sb, pc, sc,
                     self._flat(D, heads, _F32, "D"), self._flat(dt_bias, heads, _F32, "dt_bias"),
                     self._flat(state, ns * inner * d_state, _F32, "state"), ns,
                     self._flat(slots, seqs, _I32, "slots"), self._flat(has_state, seqs, _U8, "has_state"),
                     self._flat(cu_seqlens, seqs + 1, _I32, "cu_seqlens"), seqs, py, sy, code, tokens, heads,
                     head_dim, groups, d_state, ptr(scratch), nb)

    def ssm_token(self, out, xbc, dt, conv_w, conv_bias, conv_state, A, D, dt_bias, state, seqs: int,
                  heads: int, head_dim: int, groups: int, d_state: int, width: int, z=None, norm_w=None,
                  eps: float = 1e-5, slots=None, n_slots=None, dtype=None) -> None:
        """One token of each sequence through conv1d_prompt's convolution, ssm_prompt's
        scan and gated_norm (z None: no gate, norm_w None: no norm), in one
        launch; conv_state and state are updated in place.  A sequence whose
        slot is outside the arrays starts from zero and stores nothing."""
        if (seqs | heads | head_dim | groups | d_state | width) >> 31:
            _fit(seqs, heads, head_dim, groups, d_state, width)
        code = _type_of(out, dtype, "out")
        inner = heads * head_dim
        ch = inner + 2 * groups * d_state
        po, so = self._rows(out, seqs, inner, code, "out")
        px, sx = self._rows(xbc, seqs, ch, code, "xbc")
        pd, sd = self._rows(dt, seqs, heads, code, "dt")
        pz, sz = self._rows(z, seqs, inner, code, "z")
        ns = self._slots_of(state, inner * d_state, n_slots, "state")
        self._launch("ervf_ssm_token", px, sx, pd, sd, pz, sz, self._flat(conv_w, ch * width, _F32, "conv_w"),
                     self._flat(conv_bias, ch, _F32, "conv_bias"),
                     self._flat(conv_state, ns * (width - 1) * ch, _CODE_TYPES[code], "conv_state"),
                     self._flat(A, heads, _F32, "A"), self._flat(D, heads, _F32, "D"),
                     self._flat(dt_bias, heads, _F32, "dt_bias"), self._flat(norm_w, inner, _F32, "norm_w"), eps,
                     self._flat(state, ns * inner * d_state, _F32, "state"), ns,
                     self._flat(slots, seqs, _I32, "slots"), po, so, code, seqs, heads, head_dim, groups, d_state,
                     width)

    def gated_norm(self, out, y, z, w, tokens: int, groups: int, group_size: int, eps: float = 1e-5,
                   dtype=None) -> None:
        """out = w g / sqrt(mean(g^2) + eps) with g = y silu(z) (z None: y), the mean per
        group of channels.  out may be y or z itself."""
        if (tokens | groups | group_size) >> 31:
            _fit(tokens, groups, group_size)
        code = _type_of(out, dtype, "out")
        n = groups * group_size
        po, so = self._rows(out, tokens, n, code, "out")
        py, sy = self._rows(y, tokens, n, code, "y")
        pz, sz = self._rows(z, tokens, n, code, "z")
        self._launch("ervf_gated_norm", py, sy, pz, sz, self._flat(w, n, _F32, "w"), eps, po, so, code, tokens,
                     groups, group_size)

    def _scratch(self, nbytes: int):
        """Per-call scratch from torch's allocator, on the stream of the launch."""
        if not nbytes:
            return None
        if self.stream is None:
            return torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        stream = self.stream
        if not isinstance(stream, torch.cuda.Stream):
            handle = current_stream(stream, self.device)
            stream = torch.cuda.ExternalStream(handle, self.device) if handle else \
                torch.cuda.default_stream(self.device)
        with torch.cuda.stream(stream):
            return torch.empty(nbytes, dtype=torch.uint8, device=self.device)
