"""The 8-bit decoder operators on torch tensors.

    quantize_fp8, quantize_fp8_weight   casts to 8 bits with a scale per block of 128
    fp8_linear                          the product of two such operands
    block_norm                          norm, gate, residual add and the next norm in one pass
    RotaryPlan, rotary                  rotary positions on query and key heads
    token_logprobs                      log probabilities over the vocabulary, entropy, alternatives

Thin bindings of `include/vdexec_kernels.h`, which states the formulas: each
call checks its tensors, allocates its outputs where none are given, enqueues
one kernel on the current stream of the tensors' device and returns without
waiting.  Wrong arguments raise ValueError (or VdError with the library's
message) before anything runs.  Forward only: tensors that require a gradient
are refused while gradients are enabled.
"""

from __future__ import annotations

import ctypes
import threading
from typing import NamedTuple, Optional

import torch

from . import _abi

ACTIVATIONS = {"none": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "silu": 4}
FP8 = torch.float8_e4m3fn
BLOCK = 128
MAX_NORM_COLS = 16384
MAX_TOP = 64

_DTYPES = {torch.float16: _abi.VDK_FP16, torch.bfloat16: _abi.VDK_BF16, torch.float32: _abi.VDK_FP32}
_local = threading.local()
_status: dict = {}
_status_lock = threading.Lock()


def _call(name: str, device: torch.device, *args) -> None:
    err = getattr(_local, "err", None)
    if err is None:
        err = _local.err = ctypes.create_string_buffer(512)
    fn = getattr(_abi.load(), name)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream, err, 512)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream, err, 512)
    if rc:
        _abi.check(rc, err)


def _tensor(t, name: str, dims: int, dtypes=_DTYPES, device: Optional[torch.device] = None, strided: bool = True):
    """Checks one argument; `strided`: rows may lie apart, elements of a row may not."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} has dtype {t.dtype}, expected one of {[str(d) for d in dtypes]}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: this operator has no backward pass")
    if strided:
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} needs unit stride along its last dimension")
    elif not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _ld(t: torch.Tensor) -> int:
    """Row stride of a matrix; a single row has whatever stride its width needs."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _ld16(t: torch.Tensor) -> int:
    """Row stride of an 8-bit operand: a single row's may be rounded up to 16 bytes freely."""
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16


def _distinct_rows(t: torch.Tensor, name: str) -> None:
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"rows of {name} overlap")


def _output(out, shape, dtype, device, name: str) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _tensor(out, name, len(shape), (dtype,), device)
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(out.shape)}, expected {tuple(shape)}")
    _distinct_rows(out, name)
    return out


def _empty_fp8(rows: int, cols: int, device) -> torch.Tensor:
    """An 8-bit matrix whose rows start on 16-byte boundaries, as fp8_linear takes it."""
    ld = (cols + 15) // 16 * 16
    q = torch.empty(rows, ld, dtype=FP8, device=device)
    return q if ld == cols else q[:, :cols]


# ---------------------------------------------------------------------------
# 8-bit operands and their product
# ---------------------------------------------------------------------------
def quantize_fp8(x: torch.Tensor, gate: Optional[torch.Tensor] = None, act: str = "none"):
    """(q, scale): x, or act(gate) * x, as e4m3 [rows, cols] with fp32 scales [rows, ceil(cols / 128)]."""
    _tensor(x, "x", 2)
    dev = x.device
    rows, cols = x.shape
    if act not in ACTIVATIONS:
        raise ValueError(f"unknown activation {act!r}; known: {sorted(ACTIVATIONS)}")
    if gate is not None:
        _tensor(gate, "gate", 2, (x.dtype,), dev)
        if gate.shape != x.shape:
            raise ValueError(f"gate has shape {tuple(gate.shape)}, expected {tuple(x.shape)}")
    elif act != "none":
        raise ValueError("an activation needs a gate")
    if cols < 1:
        raise ValueError("x needs at least one column")
    q = _empty_fp8(rows, cols, dev)
    blocks = (cols + 127) // 128
    scale = torch.empty(rows, blocks, dtype=torch.float32, device=dev)
    if rows:
        _call("vdk_quantize_fp8", dev, x.data_ptr(), _ld(x), gate.data_ptr() if gate is not None else None,
              _ld(gate) if gate is not None else 0, ACTIVATIONS[act], rows, cols, _DTYPES[x.dtype], q.data_ptr(),
              _ld16(q), scale.data_ptr(), blocks)
    return q, scale


def quantize_fp8_weight(w: torch.Tensor):
    """(q, scale): w as e4m3 [rows, cols] with an fp32 scale per 128 x 128 block."""
    _tensor(w, "w", 2)
    rows, cols = w.shape
    if rows < 1 or cols < 1:
        raise ValueError("w needs at least one row and one column")
    q = _empty_fp8(rows, cols, w.device)
    kb = (cols + 127) // 128
    scale = torch.empty((rows + 127) // 128, kb, dtype=torch.float32, device=w.device)
    _call("vdk_quantize_fp8_weight", w.device, w.data_ptr(), _ld(w), rows, cols, _DTYPES[w.dtype], q.data_ptr(),
          _ld16(q), scale.data_ptr(), kb)
    return q, scale


def _status_word(device: torch.device) -> torch.Tensor:
    word = _status.get(device.index)
    if word is None:
        with _status_lock:
            word = _status.get(device.index)
            if word is None:
                word = torch.zeros(1, dtype=torch.int32, device=device)
                torch.cuda.synchronize(device)  # zero before any stream's kernel sees it
                _status[device.index] = word
    return word


def check_status(device=None) -> None:
    """Waits for the device and raises VdError if a pipeline wait of an earlier fp8_linear on it ran out."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    torch.cuda.synchronize(index)
    word = _status.get(index)
    if word is not None:
        code = int(word.item())
        if code:
            word.zero_()
            torch.cuda.synchronize(index)
            raise _abi.VdError(_abi.VD_ECUDA, f"a kernel reported device error {code}")


def fp8_linear(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
               bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a @ w.T + bias: a e4m3 [M, K] with scales [M, ceil(K / 128)], w e4m3 [N, K] with scales
    [ceil(N / 128), ceil(K / 128)]; out [M, N] of out_dtype.  Rows of a and w start on 16-byte boundaries (as the
    casts lay them out)."""
    _tensor(a, "a", 2, (FP8,))
    dev = a.device
    _tensor(w, "w", 2, (FP8,), dev)
    m, k = a.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"a has {k} columns and w {w.shape[1]}")
    if k < 1 or n < 1:
        raise ValueError("a and w need at least one column and w one row")
    kb = (k + 127) // 128
    for t, name, rows in ((a_scale, "a_scale", m), (w_scale, "w_scale", (n + 127) // 128)):
        _tensor(t, name, 2, (torch.float32,), dev)
        if t.shape[0] != rows or t.shape[1] != kb:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {(rows, kb)}")
    if bias is not None:
        _tensor(bias, "bias", 1, (torch.float32,), dev, strided=False)
        if bias.shape[0] != n:
            raise ValueError(f"bias has {bias.shape[0]} entries, expected {n}")
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype must be one of {[str(d) for d in _DTYPES]}")
    out = _output(out, (m, n), out_dtype, dev, "out")
    if m:
        _call("vdk_fp8_linear", dev, a.data_ptr(), _ld16(a), a_scale.data_ptr(), _ld(a_scale), w.data_ptr(), _ld16(w),
              w_scale.data_ptr(), _ld(w_scale), m, n, k, bias.data_ptr() if bias is not None else None,
              out.data_ptr(), _ld(out), _DTYPES[out_dtype], _status_word(dev).data_ptr())
    return out


# ---------------------------------------------------------------------------
# Norms around a block
# ---------------------------------------------------------------------------
class BlockNorm(NamedTuple):
    residual: torch.Tensor
    out: Optional[torch.Tensor]
    scale: Optional[torch.Tensor]


def block_norm(y: Optional[torch.Tensor], residual: Optional[torch.Tensor], post_gain: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, block_scale: float = 1.0,
               pre_gain: Optional[torch.Tensor] = None, eps: float = 1e-6, plus_one: bool = False,
               out_dtype: Optional[torch.dtype] = None, in_place: bool = False) -> BlockNorm:
    """The step between two blocks:
        u = rmsnorm(y) * post_gain            (y itself without post_gain)
        residual' = residual_scale * residual + block_scale * gate * u
        out = rmsnorm(residual') * pre_gain   (none without pre_gain)
    y [rows, cols] is the block's output (None: only the residual's norm), residual is fp32 or of y's type (None:
    zero; the new one is then fp32), gate [cols], [rows, 1], [1, cols] or [rows, cols].  out_dtype: fp16, bf16, fp32
    or float8_e4m3fn (with `scale`); y's type by default.  in_place: the new residual replaces the old one."""
    x = y if y is not None else residual
    _tensor(x, "y" if y is not None else "residual", 2)
    dev = x.device
    rows, cols = x.shape
    if not 1 <= cols <= MAX_NORM_COLS:
        raise ValueError(f"rows have {cols} columns, supported: 1 to {MAX_NORM_COLS}")
    if residual is not None:
        types = _DTYPES if y is None else (torch.float32, y.dtype)
        _tensor(residual, "residual", 2, types, dev)
        if residual.shape != x.shape:
            raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {tuple(x.shape)}")
        _distinct_rows(residual, "residual")
    elif in_place:
        raise ValueError("in_place needs a residual")
    h_dtype = torch.float32 if residual is None else residual.dtype
    y_dtype = h_dtype if y is None else y.dtype
    for g, name in ((post_gain, "post_gain"), (pre_gain, "pre_gain")):
        if g is not None:
            _tensor(g, name, 1, (torch.float32,), dev, strided=False)
            if g.shape[0] != cols:
                raise ValueError(f"{name} has {g.shape[0]} entries, expected {cols}")
    if y is None and (post_gain is not None or gate is not None):
        raise ValueError("post_gain and gate need y")
    gate_ptr, gate_type, gate_row, gate_col = None, 0, 0, 0
    if gate is not None:
        if not isinstance(gate, torch.Tensor) or gate.dim() not in (1, 2):
            raise ValueError("gate must be a tensor of 1 or 2 dimensions")
        _tensor(gate, "gate", gate.dim(), (torch.float32, y_dtype), dev)
        g2 = gate if gate.dim() == 2 else gate.unsqueeze(0)
        if g2.shape[0] not in (1, rows) or g2.shape[1] not in (1, cols):
            raise ValueError(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(x.shape)}")
        gate_ptr, gate_type = gate.data_ptr(), _DTYPES[gate.dtype]
        gate_row = g2.stride(0) if g2.shape[0] > 1 else 0
        gate_col = 1 if g2.shape[1] > 1 else 0
    if pre_gain is None:
        if out_dtype is not None:
            raise ValueError("out_dtype needs pre_gain")
    else:
        out_dtype = out_dtype or y_dtype
        if out_dtype is not FP8 and out_dtype not in _DTYPES:
            raise ValueError(f"out_dtype {out_dtype} is not supported")
    # Without a block output and with nothing to scale, the residual stays as it is.
    keep = y is None and residual is not None and residual_scale == 1.0
    if keep or in_place:
        new = residual
    else:
        new = torch.empty(rows, cols, dtype=h_dtype, device=dev)
    z = scale = None
    if pre_gain is not None:
        if out_dtype is FP8:
            z = _empty_fp8(rows, cols, dev)
            scale = torch.empty(rows, (cols + 127) // 128, dtype=torch.float32, device=dev)
        else:
            z = torch.empty(rows, cols, dtype=out_dtype, device=dev)
    if rows and (z is not None or not keep):
        _call("vdk_block_norm", dev, y.data_ptr() if y is not None else None, _ld(y) if y is not None else 0,
              _DTYPES[y_dtype], residual.data_ptr() if residual is not None else None,
              _ld(residual) if residual is not None else 0, _DTYPES[h_dtype],
              post_gain.data_ptr() if post_gain is not None else None, gate_ptr, gate_type, gate_row, gate_col,
              residual_scale, block_scale, pre_gain.data_ptr() if pre_gain is not None else None, eps, int(plus_one),
              rows, cols, None if keep else new.data_ptr(), 0 if keep else _ld(new),
              z.data_ptr() if z is not None else None, 0 if z is None else _ld16(z) if scale is not None else _ld(z),
              0 if z is None else _abi.VDK_FP8 if scale is not None else _DTYPES[out_dtype],
              scale.data_ptr() if scale is not None else None, scale.shape[1] if scale is not None else 0)
    return BlockNorm(new, z, scale)


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
class RotaryPlan:
    """The frequencies of a model's rotary positions, on one device.

    layout: "half" pairs column i with i + rotary_dim / 2, "interleaved" 2i with 2i + 1; rotary_dim (default: the
    whole head) leading columns turn.  scaling: None, or a dict with "type":
        linear   factor
        ntk      factor
        yarn     factor, original_max_position, beta_fast (32), beta_slow (1), attention_factor (0.1 ln(factor) + 1)
        llama3   factor, original_max_position, low_freq_factor, high_freq_factor
        divisors divisors (one per pair), attention_factor (1)
    """

    _TYPES = {"linear": 1, "ntk": 2, "yarn": 3, "llama3": 4, "divisors": 5}
    _KEYS = {
        "linear": (("factor", None),),
        "ntk": (("factor", None),),
        "yarn": (("factor", None), ("original_max_position", None), ("beta_fast", 32.0), ("beta_slow", 1.0),
                 ("attention_factor", 0.0)),
        "llama3": (("factor", None), ("original_max_position", None), ("low_freq_factor", None),
                   ("high_freq_factor", None)),
        "divisors": (("attention_factor", 1.0),),
    }

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, theta: float = 1e4,
                 scaling: Optional[dict] = None, layout: str = "half", device=None):
        self.head_dim = head_dim
        self.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in ("half", "interleaved"):
            raise ValueError('layout must be "half" or "interleaved"')
        self.interleaved = layout == "interleaved"
        turns, self.factor = rotary_turns(self.rotary_dim, theta, scaling)
        if self.rotary_dim > head_dim:
            raise ValueError(f"rotary_dim {self.rotary_dim} exceeds head_dim {head_dim}")
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.turns = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64,
                                  device=self.device)


def rotary_turns(rotary_dim: int, theta: float = 1e4, scaling: Optional[dict] = None):
    """(turns, factor): each pair's turns per position * 2^64 as an integer, and the factor on rotated values."""
    kind, args, divisors = 0, [], None
    if scaling is not None:
        scaling = dict(scaling)
        name = scaling.pop("type", None)
        if name not in RotaryPlan._TYPES:
            raise ValueError(f"unknown rotary scaling {name!r}; known: {sorted(RotaryPlan._TYPES)}")
        kind = RotaryPlan._TYPES[name]
        for key, default in RotaryPlan._KEYS[name]:
            value = scaling.pop(key, default)
            if value is None:
                raise ValueError(f"rotary scaling {name!r} needs {key!r}")
            args.append(float(value))
        if name == "divisors":
            divisors = [float(d) for d in scaling.pop("divisors", ())]
            if len(divisors) != rotary_dim // 2:
                raise ValueError(f"rotary scaling 'divisors' needs {rotary_dim // 2} divisors, got {len(divisors)}")
        if scaling:
            raise ValueError(f"unknown keys for rotary scaling {name!r}: {sorted(scaling)}")
    if not isinstance(rotary_dim, int) or not 2 <= rotary_dim <= 1024 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even, from 2 to 1024")
    turns = (ctypes.c_uint64 * (rotary_dim // 2))()
    factor = ctypes.c_float()
    err = ctypes.create_string_buffer(512)
    rc = _abi.load().vdk_rotary_turns(
        theta, rotary_dim, kind, (ctypes.c_double * len(args))(*args) if args else None,
        (ctypes.c_double * len(divisors))(*divisors) if divisors else None, turns, ctypes.byref(factor), err, 512)
    _abi.check(rc, err)
    return list(turns), factor.value


def _heads(x, out, name: str, plan: RotaryPlan, dtype, device):
    _tensor(x, name, 3, (dtype,) if dtype is not None else _DTYPES, device)
    if x.shape[2] != plan.head_dim:
        raise ValueError(f"{name} has head_dim {x.shape[2]}, the plan {plan.head_dim}")
    if x.shape[1] < 1:
        raise ValueError(f"{name} has no heads")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _tensor(out, name + "_out", 3, (x.dtype,), x.device)
        if out.shape != x.shape:
            raise ValueError(f"{name}_out has shape {tuple(out.shape)}, expected {tuple(x.shape)}")
    return _abi.VdkRotaryHeads(x.data_ptr(), out.data_ptr(), x.stride(0), x.stride(1), out.stride(0), out.stride(1),
                              x.shape[1]), out


def rotary(q: Optional[torch.Tensor], k: Optional[torch.Tensor], positions, plan: RotaryPlan, inverse: bool = False,
           q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None):
    """(q, k) rotated: [tokens, heads, head_dim] each (either may be None), read with any token and head strides.
    positions: int32 or int64 [tokens], or an int, the first token's position.  inverse: rotated back.  q_out /
    k_out: where to write (q / k themselves rotate in place)."""
    x = q if q is not None else k
    if x is None:
        raise ValueError("need q or k")
    _tensor(x, "q" if q is not None else "k", 3)
    tokens, dev = x.shape[0], x.device
    if plan.device != dev:
        raise ValueError(f"the plan is on {plan.device}, q and k on {dev}")
    qh = kh = None
    if q is not None:
        qh, q_out = _heads(q, q_out, "q", plan, x.dtype, dev)
    if k is not None:
        kh, k_out = _heads(k, k_out, "k", plan, x.dtype, dev)
        if k.shape[0] != tokens:
            raise ValueError(f"q has {tokens} tokens and k {k.shape[0]}")
    pos_ptr, bits, first = None, 0, 0
    if isinstance(positions, int):
        first = positions
    else:
        _tensor(positions, "positions", 1, (torch.int32, torch.int64), dev, strided=False)
        if positions.shape[0] != tokens:
            raise ValueError(f"positions has {positions.shape[0]} entries, expected {tokens}")
        pos_ptr, bits = positions.data_ptr(), 32 if positions.dtype == torch.int32 else 64
    if tokens:
        _call("vdk_rotary", dev, qh, kh, tokens, plan.head_dim, plan.rotary_dim, _DTYPES[x.dtype],
              int(plan.interleaved), int(inverse), pos_ptr, bits, first, plan.turns.data_ptr(), plan.factor)
    return q_out, k_out


# ---------------------------------------------------------------------------
# Log probabilities
# ---------------------------------------------------------------------------
class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]      # [rows, n] of the given ids
    entropy: torch.Tensor                 # [rows], in nats
    lse: torch.Tensor                     # [rows]
    top_ids: Optional[torch.Tensor]       # [rows, top] int32, -1 past the last live entry
    top_logprobs: Optional[torch.Tensor]  # [rows, top]


def token_logprobs(logits: torch.Tensor, ids: Optional[torch.Tensor] = None, top: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities of ids (int64 [rows, n] or [rows]; a negative id gives 0) under softmax(logits /
    temperature) over the whole vocabulary, the distribution's entropy and its `top` (at most 64) likeliest entries,
    equal ones by id.  logits [rows, vocab] fp16, bf16 or fp32; -inf masks an entry."""
    _tensor(logits, "logits", 2)
    dev = logits.device
    rows, vocab = logits.shape
    if vocab < 1:
        raise ValueError("logits need at least one column")
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be from 0 to {MAX_TOP}")
    n = 0
    lp = None
    if ids is not None:
        if not isinstance(ids, torch.Tensor) or ids.dim() not in (1, 2):
            raise ValueError("ids must be a tensor of 1 or 2 dimensions")
        _tensor(ids, "ids", ids.dim(), (torch.int64,), dev, strided=False)
        if ids.shape[0] != rows:
            raise ValueError(f"ids has {ids.shape[0]} rows, expected {rows}")
        n = ids.shape[1] if ids.dim() == 2 else 1
        lp = torch.empty(ids.shape, dtype=torch.float32, device=dev)
    stats = torch.empty(2, rows, dtype=torch.float32, device=dev)
    entropy, lse = stats[0], stats[1]
    top_ids = top_lp = None
    if top:
        top_ids = torch.empty(rows, top, dtype=torch.int32, device=dev)
        top_lp = torch.empty(rows, top, dtype=torch.float32, device=dev)
    if rows:
        _call("vdk_token_logprobs", dev, logits.data_ptr(), _ld(logits), rows, vocab, _DTYPES[logits.dtype],
              temperature, ids.data_ptr() if n else None, n, top, lp.data_ptr() if n else None, entropy.data_ptr(),
              lse.data_ptr(), top_ids.data_ptr() if top else None, top_lp.data_ptr() if top else None)
    return TokenLogprobs(lp, entropy, lse, top_ids, top_lp)
