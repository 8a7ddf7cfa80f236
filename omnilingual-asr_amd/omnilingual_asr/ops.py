"""Operators on torch tensors: checked arguments, buffers from torch's allocator, the tensors' own device and its current
stream.  Each call is one or two launches of liboasr_hip.so (the C ABI takes raw pointers: include/oasr.h); nothing
synchronises, so a call may be captured into a HIP graph.  A mistake raises ValueError before anything is launched.

No counterpart in the reference, whose projections and answers are made by a remote model
(ref:src/omnilingual_asr/models/inference/gemini_pipeline.py:512-530).
"""

from __future__ import annotations

import math
import numbers
import operator
from typing import NamedTuple

import torch

from . import _hip
from .weights import quantize_rows_i8

EPILOGUES = {"bias": _hip.EPI_BIAS_BF16, "swish": _hip.EPI_BIAS_SWISH_BF16, "glu": _hip.EPI_GLU_BF16,
             "residual": _hip.EPI_RESIDUAL_F32, "float": _hip.EPI_BIAS_F32}
_INT8, _FLOAT32, _BFLOAT16, _LOGITS = (torch.int8,), (torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)
_NORM_WIDTHS = (256, 512, 1024, 2048, 4096)
_EINVAL = -1                                             # OASR_EINVAL: refused before a launch


def _call(name: str, device: torch.device, *args) -> None:
    """One C call on `device`'s current stream; the device is made the current one where it is not."""
    fn = getattr(_hip.lib(), name)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, _hip.stream_ptr(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _hip.stream_ptr(device.index))
    if rc:
        if rc == _EINVAL:
            raise ValueError(_hip.lib().oasr_last_error().decode("utf-8", "replace"))
        _hip.check(rc, name)


def _number(v, what: str) -> float:
    if type(v) is float:
        return v
    if not isinstance(v, numbers.Real):                  # a tensor among them: its value is on the device
        raise ValueError(f"{what} must be a number")
    return float(v)


def _integer(v, what: str) -> int:
    if type(v) is int:
        return v
    if isinstance(v, torch.Tensor) or not hasattr(v, "__index__"):
        raise ValueError(f"{what} must be an integer")
    return operator.index(v)


def _rows(t, what: str, dtypes: tuple):
    """(tensor, rows, columns, row pitch) of a [..., columns] tensor whose rows are contiguous and evenly spaced."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise ValueError(f"{what} must be a tensor of {' or '.join(map(str, dtypes))}")
    if not t.is_cuda:
        raise ValueError(f"{what} must be on a HIP device; there is no CPU fallback")
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{what} must have at least one column")
    cols = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // cols, cols, cols
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), cols)
    rows = t.shape[0]
    pitch = t.stride(0) if rows > 1 else cols
    if cols > 1 and t.stride(1) != 1 or pitch < cols:
        raise ValueError(f"{what} must have contiguous rows that do not overlap")
    return t, rows, cols, pitch


def _overlap(a, b) -> bool:
    """Whether the memory between the first and the last element of two strided tensors meets."""
    def span(t):
        if t.numel() == 0:
            return 0, 0
        lo = t.data_ptr()
        return lo, lo + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _vector(t, n: int, what: str, device) -> int | None:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{what} must be a contiguous float32 vector of {n} on {device}")
    return t.data_ptr()


class LinearI8:
    """y = epilogue(x W^T + bias) with W and x in 8-bit integers: W has one scale per output row, every row of x gets its
    own (max|row| / 127) inside the call, and the products are summed exactly in 32-bit integers.

    `epilogue`: "bias" -> bf16, "swish" -> bf16, "glu" -> bf16 of half the width (rows of W interleaved as
    `weights.glu_interleave` does, a multiple of 32), "float" -> float32, "residual" -> resid + alpha * (...) in float32.
    Forward only: results carry no gradient.  The layer owns what it reads: the weights are packed and scale and bias copied on
    the stream that is current when the object is made, so a module they came from may be moved, changed or dropped afterwards.
    A call on another stream has to wait for that one, as for any tensor made there, and the object must not be in use by
    another stream when it is dropped.  `scale`, `bias` and `packed` give the layer's own memory and cannot be assigned.
    A layer can be copied (copy.deepcopy) and pickled; it has to be on a HIP device when it is loaded."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None):
        """`weight`: float [out, in] on a HIP device; quantised per output row."""
        if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not weight.is_floating_point():
            raise ValueError("weight must be a float tensor [out, in]")
        if weight.shape[1] < 1:
            raise ValueError("weight must have at least one column")
        self._lay_out(*quantize_rows_i8(weight.detach()), bias)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None) -> "LinearI8":
        """From int8 codes [out, in] and float32 scales [out] (weight = codes * scale[:, None])."""
        self = cls.__new__(cls)
        self._lay_out(codes, scale, bias)
        return self

    def _lay_out(self, codes, scale, bias):
        if not isinstance(codes, torch.Tensor) or codes.dim() != 2:
            raise ValueError("codes must be [out, in]")
        codes, n, k, ldw = _rows(codes, "codes", _INT8)
        if n < 1 or not 1 <= k <= 131072:
            raise ValueError("a weight has at least one row and 1 to 131072 columns")
        self.device, self.out_features, self.in_features = codes.device, n, k
        _vector(scale, n, "scale", codes.device), _vector(bias, n, "bias", codes.device)
        if scale is None:
            raise ValueError("scale must be given")
        packed = codes.new_empty((int(_hip.lib().oasr_gemm_i8_packed_bytes(n, k)),))
        _call("oasr_gemm_pack_w_i8", self.device, codes.data_ptr(), ldw, n, k, packed.data_ptr())
        self._own(packed, scale.detach().clone(), None if bias is None else bias.detach().clone())

    def _own(self, packed, scale, bias):
        """The layer's own buffers and their addresses, which hold as long as nobody else can replace a buffer's storage: a
        Parameter's is replaced in place by Module.to() and the like, the tensor object staying the same."""
        self._packed, self._scale, self._bias = packed, scale, bias
        self._packed_ptr, self._scale_ptr = packed.data_ptr(), scale.data_ptr()
        self._bias_ptr = None if bias is None else bias.data_ptr()

    def __getstate__(self):
        return {"packed": self._packed, "scale": self._scale, "bias": self._bias, "shape": (self.out_features, self.in_features)}

    def __setstate__(self, state):
        """A copy or an unpickled layer reads its own buffers, on the device on which they are now."""
        (n, k), packed, scale, bias = state["shape"], state["packed"], state["scale"], state["bias"]
        _rows(packed, "packed weights", _INT8)
        if packed.shape != (int(_hip.lib().oasr_gemm_i8_packed_bytes(n, k)),):
            raise ValueError(f"packed weights are not those of a layer [{n}, {k}]")
        self.device, self.out_features, self.in_features = packed.device, n, k
        _vector(scale, n, "scale", packed.device), _vector(bias, n, "bias", packed.device)
        self._own(packed, scale, bias)

    @property
    def packed(self) -> torch.Tensor:
        return self._packed.detach()

    @property
    def scale(self) -> torch.Tensor:
        return self._scale.detach()

    @property
    def bias(self) -> torch.Tensor | None:
        return None if self._bias is None else self._bias.detach()

    def _output(self, x, epilogue, resid, out):
        """(epilogue code, output, its row pitch, residual's pointer, its row pitch) for input x."""
        epi = EPILOGUES.get(epilogue) if isinstance(epilogue, str) else None
        if epi is None:
            raise ValueError(f"epilogue must be one of {', '.join(EPILOGUES)}")
        n = self.out_features
        if epi == _hip.EPI_GLU_BF16:
            if n % 32:
                raise ValueError("the GLU epilogue needs a multiple of 32 output rows")
            n //= 2
        dtype = torch.float32 if epi >= _hip.EPI_RESIDUAL_F32 else torch.bfloat16
        shape = (*x.shape[:-1], n)
        given = out is not None
        if not given:
            out = x.new_empty(shape, dtype=dtype)
            if epi != _hip.EPI_RESIDUAL_F32 and resid is None:
                return epi, out, n, None, 0
        elif not isinstance(out, torch.Tensor) or out.shape != shape or out.device != self.device:
            raise ValueError(f"out must be of shape {shape} on {self.device}")
        flat, _, _, ldc = _rows(out, "out", (dtype,))
        if given and flat.data_ptr() != out.data_ptr():
            raise ValueError("out must have evenly spaced rows")
        if given and _overlap(flat, x):
            raise ValueError("out must not overlap x")
        if epi != _hip.EPI_RESIDUAL_F32:
            if resid is not None:
                raise ValueError("resid goes with the residual epilogue only")
            return epi, out, ldc, None, 0
        if not isinstance(resid, torch.Tensor) or resid.shape != shape or resid.device != self.device:
            raise ValueError(f"the residual epilogue needs resid of shape {shape} on {self.device}")
        r, _, _, ldr = _rows(resid, "resid", _FLOAT32)
        if given and _overlap(flat, r) and (r.data_ptr() != flat.data_ptr() or ldr != ldc):
            raise ValueError("resid may be out itself, or must not overlap it")
        return epi, out, ldc, r, ldr

    def __call__(self, x: torch.Tensor, *, epilogue: str = "bias", resid: torch.Tensor | None = None, alpha: float = 1.0,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """x bf16 [..., in] -> [..., out].  `out` may be given (rows evenly spaced) and may be `resid`."""
        x2, m, k, ldx = _rows(x, "x", _BFLOAT16)
        if k != self.in_features or x.device != self.device:
            raise ValueError(f"x must have {self.in_features} columns on {self.device}")
        alpha = _number(alpha, "alpha")
        epi, out, ldc, resid, ldr = self._output(x, epilogue, resid, out)
        if m == 0:
            return out
        ws_bytes = _hip.lib().oasr_linear_i8_workspace_bytes(m, self.out_features, k)
        ws = x.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
        _call("oasr_linear_i8", self.device, x2.data_ptr(), ldx, self._packed_ptr, self._scale_ptr, self._bias_ptr,
              None if resid is None else resid.data_ptr(), ldr, out.data_ptr(), ldc, m, self.out_features, k, alpha, epi,
              None if ws is None else ws.data_ptr(), ws_bytes)
        return out

    def normed(self, x: torch.Tensor, gain: torch.Tensor, shift: torch.Tensor, *, eps: float = 1e-5, epilogue: str = "bias",
               resid: torch.Tensor | None = None, alpha: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
        """The layer on LayerNorm(x) * gain + shift: x float32 [..., in] contiguous, in 256, 512, 1024, 2048 or 4096.  The
        normalised rows go to 8-bit integers without being stored in between."""
        x2, m, k, ldx = _rows(x, "x", _FLOAT32)
        if k != self.in_features or x.device != self.device:
            raise ValueError(f"x must have {self.in_features} columns on {self.device}")
        if k not in _NORM_WIDTHS or ldx != k or x2.data_ptr() % 16:
            raise ValueError(f"normed takes contiguous, 16-byte aligned rows of {', '.join(map(str, _NORM_WIDTHS))} columns")
        gain_ptr, shift_ptr = _vector(gain, k, "gain", self.device), _vector(shift, k, "shift", self.device)
        if gain_ptr is None or shift_ptr is None or (gain_ptr | shift_ptr) % 16:
            raise ValueError("gain and shift must be given, 16-byte aligned")
        alpha, eps = _number(alpha, "alpha"), _number(eps, "eps")
        epi, out, ldc, resid, ldr = self._output(x, epilogue, resid, out)
        if m == 0:
            return out
        codes, scale = x.new_empty((m, k), dtype=torch.int8), x.new_empty((m,))
        _call("oasr_layernorm_i8", self.device, x2.data_ptr(), gain_ptr, shift_ptr, codes.data_ptr(), scale.data_ptr(), m, k, eps, 0)
        _call("oasr_gemm_i8", self.device, codes.data_ptr(), k, self._packed_ptr, scale.data_ptr(), self._scale_ptr, self._bias_ptr,
              None if resid is None else resid.data_ptr(), ldr, out.data_ptr(), ldc, m, self.out_features, k, alpha, epi)
        return out


MAX_ALTERNATIVES = 32


class TokenScores(NamedTuple):
    """What `token_scores` returns; float32 (ids int32) on the logits' device, natural logarithms."""
    logprobs: torch.Tensor      # of the given tokens
    entropy: torch.Tensor       # of each row's distribution
    ids: torch.Tensor           # [..., alternatives]: the likeliest tokens, best first, -1 where there are fewer
    best: torch.Tensor          # [..., alternatives]: their log probabilities


def _int32(t, shape, what: str, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.shape != shape or t.device != device:
        raise ValueError(f"{what} must be an int32 tensor of shape {tuple(shape)} on {device}")
    return t if t.is_contiguous() else t.contiguous()


def _score_outputs(lead, given, alternatives, like, rows, vocab, n):
    """The outputs of `rows` rows with `n` given tokens each, after the checks of sizes (the C call takes vocab, n and a batch as
    32-bit integers)."""
    if not 0 <= alternatives <= MAX_ALTERNATIVES:
        raise ValueError(f"alternatives must lie in [0, {MAX_ALTERNATIVES}]")
    if rows >= 1 << 24 or vocab >= 1 << 30 or n >= 1 << 31:
        raise ValueError("token scores take fewer than 2^24 rows, 2^30 columns and 2^31 given tokens a row")
    new, f32, listed = like.new_empty, torch.float32, (*lead, alternatives)
    return TokenScores(new(given, dtype=f32), new(lead, dtype=f32), new(listed, dtype=torch.int32), new(listed, dtype=f32))


def _score(name, z, args, out, rows, vocab, alternatives):
    """The call that both forms make: `args` between the logits' type and the outputs."""
    ws_bytes = _hip.lib().oasr_token_scores_workspace_bytes(rows, vocab, alternatives)
    ws = z.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
    _call(name, z.device, z.data_ptr(), _hip.F32 if z.dtype == torch.float32 else _hip.BF16, *args, out.logprobs.data_ptr(),
          out.entropy.data_ptr(), alternatives, out.ids.data_ptr(), out.best.data_ptr(), None if ws is None else ws.data_ptr(), ws_bytes)
    return out


def token_scores(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, alternatives: int = 0) -> TokenScores:
    """Log probabilities of given tokens under rows of logits [..., vocab] (float32 or bfloat16; rows evenly spaced), with
    every row's entropy and its `alternatives` likeliest tokens.  `tokens`: int32 [...] or [..., n]; a negative one means
    none (0).  Masked logits (-inf) have probability 0 and are no alternatives; include/oasr.h says what else rows hold."""
    z, rows, vocab, ld = _rows(logits, "logits", _LOGITS)
    alternatives = _integer(alternatives, "alternatives")
    lead, device = logits.shape[:-1], logits.device
    given, n = (*lead, 0), 0
    if tokens is not None:
        given = tokens.shape if isinstance(tokens, torch.Tensor) else ()
        if given != lead and given[:-1] != lead:
            raise ValueError(f"tokens must be of shape {tuple(lead)} or {tuple(lead)} and one more dimension")
        tokens, n = _int32(tokens, given, "tokens", device), 1 if given == lead else given[-1]
    out = _score_outputs(lead, given, alternatives, logits, rows, vocab, n)
    if rows == 0:
        return out
    return _score("oasr_token_scores", z, (ld, rows, vocab, None if tokens is None else tokens.data_ptr(), n), out, rows, vocab,
                  alternatives)


def ctc_token_scores(logits: torch.Tensor, tokens: torch.Tensor, frames: torch.Tensor, *, vocab: int | None = None,
                     alternatives: int = 0) -> TokenScores:
    """The same for the tokens a CTC decode emitted: logits [batch, frames, pitch] of which the first `vocab` columns count
    (all by default), tokens and frames int32 [batch, n] as `HipEngine.decode` returns them (-1 past an utterance's
    count: log probability 0, entropy 0, no alternatives)."""
    if not isinstance(logits, torch.Tensor) or logits.dim() != 3 or not logits.is_contiguous():
        raise ValueError("logits must be a contiguous tensor [batch, frames, pitch]")
    batch, t_pad, ld = logits.shape
    _rows(logits, "logits", _LOGITS)
    vocab, alternatives = ld if vocab is None else _integer(vocab, "vocab"), _integer(alternatives, "alternatives")
    if not 1 <= vocab <= ld:
        raise ValueError(f"vocab must lie in [1, {ld}]")
    if not isinstance(tokens, torch.Tensor) or tokens.dim() != 2 or tokens.shape[0] != batch:
        raise ValueError("tokens must be [batch, n]")
    device, shape = logits.device, tokens.shape
    tokens, frames = _int32(tokens, shape, "tokens", device), _int32(frames, shape, "frames", device)
    if t_pad == 0 and tokens.numel():
        raise ValueError("logits have no frames")
    out = _score_outputs(shape, shape, alternatives, logits, tokens.numel(), vocab, 1)
    if tokens.numel() == 0:
        return out
    return _score("oasr_ctc_token_scores", logits, (ld, vocab, batch, t_pad, tokens.data_ptr(), frames.data_ptr(), shape[1]), out,
                  tokens.numel(), vocab, alternatives)
