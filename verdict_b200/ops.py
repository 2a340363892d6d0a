"""The 8-bit decoder operators on torch tensors.

    quantize_fp8, quantize_fp8_weight   casts to 8 bits with a scale per block of 128
    fp8_linear                          the product of two such operands
    block_norm                          norm, gate, residual add and the next norm in one pass
    RotaryPlan, rotary                  rotary positions on query and key heads
    token_logprobs                      log probabilities over the vocabulary, entropy, alternatives

Thin bindings of `include/vdexec_kernels.h`, which states the formulas, through
`csrc/torch_ops.cpp`: each call checks its tensors, allocates its outputs where
none are given, enqueues one kernel on the current stream of the tensors'
device and returns without waiting.  Wrong arguments raise ValueError (or VdError with the library's
message) before anything runs.  Forward only: tensors that require a gradient
are refused while gradients are enabled.
"""

from __future__ import annotations

import ctypes
import importlib
import threading
from typing import NamedTuple, Optional

import torch

from . import _abi
from . import build as _build


def _load():
    """The torch binding (built first where it or the library is missing or stale); it loads libvdexec.so.  A binding
    made for other C entries or another torch is never used: it would pass arguments that are read as others."""
    _abi.load()
    if not _build.library_has_this_header():
        raise RuntimeError("libvdexec.so was built from other headers and could not be rebuilt; run "
                           "`python -m verdict_b200.build`")
    if not _build.torch_up_to_date():
        _build.build_torch_ops()
    return importlib.import_module("verdict_b200._torch_ops")


_ops = _load()

ACTIVATIONS = {"none": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "silu": 4}
FP8 = torch.float8_e4m3fn
BLOCK = 128
MAX_NORM_COLS = 16384
MAX_TOP = 64

_CODES = {torch.float16: _abi.VDK_FP16, torch.bfloat16: _abi.VDK_BF16, torch.float32: _abi.VDK_FP32}
_NORM_CODES = {**_CODES, FP8: _abi.VDK_FP8, None: -1}
_status: dict = {}     # device index -> the word that fp8_linear's kernels leave a code in
_failures: dict = {}   # device index -> (how many codes check_status has found there, the last one)
_status_lock = threading.Lock()
_thread = threading.local()  # .seen: device index -> how many of those failures this thread knows of


# ---------------------------------------------------------------------------
# 8-bit operands and their product
# ---------------------------------------------------------------------------
def quantize_fp8(x: torch.Tensor, gate: Optional[torch.Tensor] = None, act: str = "none"):
    """(q, scale): x, or act(gate) * x, as e4m3 [rows, cols] with fp32 scales [rows, ceil(cols / 128)]."""
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"unknown activation {act!r}; known: {sorted(ACTIVATIONS)}")
    return _ops.quantize_fp8(x, gate, code)


def quantize_fp8_weight(w: torch.Tensor):
    """(q, scale): w as e4m3 [rows, cols] with an fp32 scale per 128 x 128 block."""
    return _ops.quantize_fp8_weight(w)


def _status_word(device: torch.device) -> torch.Tensor:
    index = device.index
    try:
        _thread.seen[index]
        return _status[index]
    except (AttributeError, KeyError):
        pass
    with _status_lock:
        word = _status.get(index)
        if word is None:
            word = torch.zeros(1, dtype=torch.int32, device=device)
            torch.cuda.synchronize(device)  # zero before any stream's kernel sees it
            _status[index] = word
        if not hasattr(_thread, "seen"):
            _thread.seen = {}
        _thread.seen.setdefault(index, _failures.get(index, (0, 0))[0])
    return word


def check_status(device=None) -> None:
    """Waits for the device and raises VdError if a pipeline wait of an earlier fp8_linear on it ran out.  Threads share
    a device: one that has called fp8_linear there learns of every such failure since its first call, once, whichever
    thread's call it was and whoever asked first."""
    index = torch.device(device).index if device is not None else None
    if index is None:
        index = torch.cuda.current_device()
    torch.cuda.synchronize(index)
    with _status_lock:
        count, code = _failures.get(index, (0, 0))
        word = _status.get(index)
        found = int(word.item()) if word is not None else 0
        if found:
            word.zero_()
            torch.cuda.synchronize(index)
            count, code = _failures[index] = (count + 1, found)
        seen = getattr(_thread, "seen", {})
        # A thread that only asks is told of what it finds itself.
        new = count > seen.get(index, count - bool(found))
        if index in seen:
            seen[index] = count
    if new:
        raise _abi.VdError(_abi.VD_ECUDA, f"a kernel reported device error {code}")


def fp8_linear(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
               bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a @ w.T + bias: a e4m3 [M, K] with scales [M, ceil(K / 128)], w e4m3 [N, K] with scales
    [ceil(N / 128), ceil(K / 128)]; out [M, N] of out_dtype.  Rows of a and w start on 16-byte boundaries (as the
    casts lay them out).  The first call on a device makes the word that check_status reads and waits for it once: make
    that call before any stream capture."""
    code = _CODES.get(out_dtype)
    if code is None:
        raise ValueError(f"out_dtype must be one of {[str(d) for d in _CODES]}")
    if not isinstance(a, torch.Tensor) or not a.is_cuda:
        raise ValueError("a must be a tensor on a CUDA device")
    return _ops.fp8_linear(a, a_scale, w, w_scale, bias, code, out, _status_word(a.device))


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
    code = _NORM_CODES.get(out_dtype)
    if code is None:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    return BlockNorm._make(_ops.block_norm(y, residual, post_gain, gate, residual_scale, block_scale, pre_gain, eps,
                                           plus_one, code, in_place))


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


def rotary(q: Optional[torch.Tensor], k: Optional[torch.Tensor], positions, plan: RotaryPlan, inverse: bool = False,
           q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None):
    """(q, k) rotated: [tokens, heads, head_dim] each (either may be None), read with any token and head strides.
    positions: int32 or int64 [tokens], or an int, the first token's position.  inverse: rotated back.  q_out /
    k_out: where to write (q / k themselves rotate in place)."""
    return _ops.rotary(q, k, positions, plan.turns, plan.head_dim, plan.rotary_dim, plan.interleaved, plan.factor,
                       inverse, q_out, k_out)


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
    return TokenLogprobs._make(_ops.token_logprobs(logits, ids, top, temperature))
