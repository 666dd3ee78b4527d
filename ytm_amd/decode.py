"""From clause outputs to an answer, on the GPU (not in the reference).

A model with many outputs, such as one a word of a vocabulary (up to 4096; more with weights from
elsewhere), answers in three steps:

    codes, scales = decode.pack_model(tm)                          # once: weights in 4 bits
    bits = decode.pack_outputs(tm.transform(X))                    # clause outputs, packed
    scores = decode.readout(bits, codes, scales, clauses=C)        # class sums (N, K)
    scores = decode.adjust_scores(scores, tokens=said, ...)        # penalties, bias, grammar
    token, logprob = decode.choose(scores, top_p=..., noise=...)   # the answer of each row

readout, adjust_scores and choose take torch tensors on one GPU and put their work on the
current stream of that GPU without waiting for it, as torch's own operations do (they may be
captured into a graph); pack_model, pack_weights and pack_outputs turn the framework's host arrays
into such tensors.  Rows may be any distance apart; a row's elements follow one another.  A wrong
argument raises TypeError or ValueError before anything is launched.  There are no gradients:
clause outputs are bits made by automata and the codes are made from trained weights, so tensors
that require a gradient, or have a tangent of forward mode, are refused.  The formulas are at
ytm_readout, ytm_adjust_scores and ytm_choose in include/ytm.h.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch
from torch.autograd import forward_ad as _forward_ad

from ._lib import DTYPE_BF16, DTYPE_BITS, DTYPE_F16, DTYPE_F32, check, lib

_FLOATS = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}
_CLAUSES = {torch.int32: DTYPE_BITS, **_FLOATS}
# E2M1 magnitudes of the codes 0..7, and the points between them
_MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], np.float32)
_BETWEEN = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])


def pack_weights(weights: np.ndarray, group: int = 32, dtype: torch.dtype = torch.float32,
                 device: str | torch.device = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """Clause weights (C, K), as get_weights() gives them, in 4 bits for readout: codes uint8
    (K, 16 ceil(C/32)) and scales (K, ceil(C/group)) of `dtype`.  A group's largest weight becomes
    6 (a code's largest value) times its scale, the others the nearest code, ties to the smaller
    magnitude; where that scale would be 0, it is the least positive one and all weights become the
    nearest code.  Weights whose scale `dtype` does not hold (in float16 those above 393000) are
    refused.  Runs on the host."""
    with np.errstate(over="ignore"):  # refused below
        w = np.asarray(weights, dtype=np.float32)
    if w.ndim != 2:
        raise ValueError("weights must have shape (clauses, outputs).")
    if not np.isfinite(w).all():
        raise ValueError("weights must be finite in float32.")
    if group < 32 or group % 32:
        raise ValueError("group must be a multiple of 32.")
    if dtype not in _FLOATS:
        raise TypeError("scales are float32, float16 or bfloat16.")
    C, K = w.shape
    groups, padded = -(-C // group), 32 * -(-C // 32)
    largest = np.zeros((K, groups), np.float32)
    for q in range(groups):
        largest[:, q] = np.abs(w[q * group:(q + 1) * group]).max(0)
    scales = torch.from_numpy(largest / 6.0).to(dtype)
    if not torch.isfinite(scales).all():
        raise ValueError(f"weights of {largest.max():g} are past what {dtype} scales hold.".replace("torch.", ""))
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    scales = torch.where(scales > 0, scales, torch.tensor(least, dtype=dtype))
    scales[torch.from_numpy(largest) == 0] = 1.0  # whatever it is, their codes are 0
    per_clause = scales.double().numpy().repeat(group, axis=1)[:, :C]
    scaled = w.T / per_clause  # in float64, so that the nearest code is
    code = np.zeros((K, padded), np.uint8)
    code[:, :C] = np.searchsorted(_BETWEEN, np.abs(scaled), side="left") | (scaled < 0).astype(np.uint8) << 3
    return torch.from_numpy(code[:, 0::2] | code[:, 1::2] << 4).to(device), scales.to(device)


def pack_model(tm, group: int = 32, dtype: torch.dtype = torch.float32,
               device: str | torch.device = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """pack_weights of a model's clause weights, for the clause outputs that transform() gives:
    clauses without literals, which transform() lets fire and class sums leave out, get zeros.
    Models with clause banks (coalesced=False) are refused."""
    if not tm.coalesced:
        raise ValueError("pack_model takes coalesced models, not clause banks.")
    weights = tm.get_weights()
    weights[~tm.get_literals().any(axis=1)] = 0.0
    return pack_weights(weights, group, dtype, device)


def unpack_weights(codes: torch.Tensor, scales: torch.Tensor, clauses: int, group: int = 32) -> np.ndarray:
    """The weights (clauses, K) float32 that codes and scales stand for.  Runs on the host."""
    c = codes.cpu().numpy()
    code = np.stack((c & 15, c >> 4), 2).reshape(c.shape[0], -1)[:, :clauses]
    value = np.where(code & 8, -1, 1).astype(np.float32) * _MAGNITUDES[code & 7]
    return (value * scales.float().cpu().numpy().repeat(group, axis=1)[:, :clauses]).T


def pack_outputs(outputs: np.ndarray, device: str | torch.device = "cuda") -> torch.Tensor:
    """Clause outputs (N, C), as transform() gives them, as bits for readout: int32
    (N, ceil(C/32)), bit b of word j = clause 32 j + b."""
    on = np.asarray(outputs) != 0
    if on.ndim != 2:
        raise ValueError("clause outputs must have shape (samples, clauses).")
    N, C = on.shape
    packed = np.zeros((N, 4 * -(-C // 32)), np.uint8)
    packed[:, :-(-C // 8)] = np.packbits(on, axis=1, bitorder="little")
    return torch.from_numpy(packed.view("<i4")).to(device)


# Operators of a few microseconds: the checks are one condition each, and what is wrong is found out
# where it fails.
_Tensor = torch.Tensor
_device_now = torch._C._cuda_getDevice
_stream_of = torch._C._cuda_getCurrentRawStream
_changed = torch._C._increment_version  # what torch.autograd.graph.increment_version calls


def _refuse(t, name: str, dims: tuple, dtype, shape: str, device: int) -> None:
    """Raises what is wrong with operand t; `shape` says what its shape must be where it does not fit.
    Nothing where t only requires a gradient and none is recorded."""
    if not isinstance(t, _Tensor):
        raise TypeError(f"{name} must be a torch tensor.")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU.")
    if device >= 0 and t.get_device() != device:
        raise ValueError(f"{name} must be on cuda:{device}, not {t.device}.")
    if t.dim() not in dims:
        raise ValueError(f"{name} must have {' or '.join(map(str, dims))} dimensions.")
    if dtype is not None and t.dtype not in (dtype if isinstance(dtype, (tuple, dict)) else (dtype,)):
        names = dtype if isinstance(dtype, (tuple, dict)) else (dtype,)
        raise TypeError(f"{name} must be {' or '.join(str(d).removeprefix('torch.') for d in names)}, not {t.dtype}.")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}'s rows must be contiguous.")
    if shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}.")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient; this operator has none.")


def _no_tangents(**operands) -> None:
    """Refuses operands whose forward-mode derivative would be dropped."""
    if torch._C._is_fwd_grad_enabled():
        for name, t in operands.items():
            if isinstance(t, _Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has a tangent; this operator has no derivative.")


def _rows_of(t, name: str, types: dict) -> tuple[int, int, int, int]:
    """(type code, rows, width, device) of an operator's first operand."""
    if not (isinstance(t, _Tensor) and t.is_cuda and t.dim() == 2 and t.dtype in types and not t.requires_grad
            and (t.stride(1) == 1 or t.shape[1] < 2)):
        _refuse(t, name, (2,), types, "", -1)
    rows, width = t.shape
    return types[t.dtype], rows, width, t.get_device()


def _matrix(t, name: str, dtype: torch.dtype, rows: int, width: int, device: int) -> tuple[int | None, int]:
    """(address, row stride; 0 for one row shared by all) of an optional operand (rows, width) or
    (width)."""
    if t is None:
        return None, 0
    if isinstance(t, _Tensor) and t.dtype is dtype and t.get_device() == device and not t.requires_grad:
        shape = t.shape
        if shape == (rows, width):
            if t.stride(1) == 1 or width < 2:
                return t.data_ptr(), t.stride(0) if rows > 1 else 0
        elif shape == (width,) and (t.stride(0) == 1 or width < 2):
            return t.data_ptr(), 0
    fits = isinstance(t, _Tensor) and tuple(t.shape) in ((rows, width), (width,))
    _refuse(t, name, (1, 2), dtype, "" if fits else f"({rows}, {width}) or ({width},)", device)
    return t.data_ptr(), t.stride(0) if t.dim() == 2 and rows > 1 else 0


def _per_row(t, name: str, dtype: torch.dtype, rows: int, device: int) -> int | None:
    if t is None:
        return None
    if not (isinstance(t, _Tensor) and t.dtype is dtype and t.get_device() == device and t.shape == (rows,)
            and (t.stride(0) == 1 or rows < 2) and not t.requires_grad):
        fits = isinstance(t, _Tensor) and tuple(t.shape) == (rows,)
        _refuse(t, name, (1,), dtype, "" if fits else f"({rows},)", device)
    return t.data_ptr()


def _result(out, shape: tuple[int, int], device: int) -> tuple[torch.Tensor, int]:
    """(the output tensor, its type code)"""
    if out is None:
        return torch.empty(shape, dtype=torch.float32, device=torch.device("cuda", device)), DTYPE_F32
    if not (isinstance(out, _Tensor) and out.get_device() == device and out.shape == shape and out.dtype in _FLOATS
            and (out.stride(1) == 1 or shape[1] < 2) and not out.requires_grad):
        fits = isinstance(out, _Tensor) and tuple(out.shape) == shape
        _refuse(out, "out", (2,), _FLOATS, "" if fits else str(shape), device)
    _changed((out,))  # for a backward pass that has kept it
    return out, _FLOATS[out.dtype]


def _call(function, device: int, *args) -> None:
    """function(*args, current stream) with `device` current."""
    if device == _device_now():
        rc = function(*args, _stream_of(device))
    else:
        with torch.cuda.device(device):
            rc = function(*args, _stream_of(device))
    if rc:
        check(rc)


def _workspace(function, device: torch.device, *args) -> tuple[int, torch.Tensor | None]:
    """The bytes that function(*args) asks for, and a tensor of them (None for 0)."""
    need = ctypes.c_int64()
    rc = function(*args, need)
    if rc:
        check(rc)
    return need.value, torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None


def readout(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, group: int = 32, clauses: int | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """Class sums (N, K) of clause outputs x through weights in 4 bits (pack_weights).

    x: bits, int32 (N, ceil(C/32)) as pack_outputs gives them, C being `clauses` (default: every
    bit); or float32, float16 or bfloat16 (N, C), outputs averaged over models or patches.
    out: where the sums go, float32, float16 or bfloat16 (default: a new float32 tensor)."""
    if _forward_ad._current_level >= 0:
        _no_tangents(x=x, scales=scales, out=out)
    x_type, N, width, device = _rows_of(x, "x", _CLAUSES)
    if x_type == DTYPE_BITS:
        C = 32 * width if clauses is None else int(clauses)
        if -(-C // 32) != width:
            raise ValueError(f"x must hold {-(-C // 32)} words of clause bits a row, not {width}.")
    else:
        C = width
        if clauses is not None and int(clauses) != C:
            raise ValueError(f"x must have {clauses} columns, not {C}.")
    group = int(group)
    if not 32 <= group < 1 << 63 or group % 32:  # the library takes 64 bits
        raise ValueError("group must be a multiple of 32.")
    if not (isinstance(codes, _Tensor) and codes.dtype is torch.uint8 and codes.get_device() == device
            and codes.dim() == 2 and (codes.stride(1) == 1 or codes.shape[1] < 2)):
        _refuse(codes, "codes", (2,), torch.uint8, "", device)
    K, held = codes.shape
    if held < 16 * -(-C // 32):
        raise ValueError(f"codes must hold {16 * -(-C // 32)} bytes an output, not {held}.")
    groups = -(-C // group)
    if not (isinstance(scales, _Tensor) and scales.dtype in _FLOATS and scales.get_device() == device
            and scales.shape == (K, groups) and (scales.stride(1) == 1 or groups < 2) and not scales.requires_grad):
        fits = isinstance(scales, _Tensor) and tuple(scales.shape) == (K, groups)
        _refuse(scales, "scales", (2,), _FLOATS, "" if fits else f"({K}, {groups})", device)
    out, out_type = _result(out, (N, K), device)
    need, workspace = 0, None
    if N > 16 or C * N > 4096:  # fewer are held in one block's LDS
        need, workspace = _workspace(lib.ytm_readout_workspace, x.device, x_type, N, C, K)
    _call(lib.ytm_readout, device, x.data_ptr(), x_type, x.stride(0), N, C, codes.data_ptr(), codes.stride(0),
          scales.data_ptr(), _FLOATS[scales.dtype], scales.stride(0), group, K, out.data_ptr(), out_type,
          out.stride(0), workspace.data_ptr() if need else None, need)
    return out


def adjust_scores(scores: torch.Tensor, tokens: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                  prompt: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                  frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Scores (N, V) shaped by what was said, by a bias and by a grammar.

    tokens: int32 (N, T), each row's history, of which the first lengths[n] entries count (int32
    (N,), default all) and the first prompt[n] of these were given, not answered (int32 (N,),
    default none).  repetition, frequency, presence: float32 (N,) penalties: an answer anywhere in
    the history has its score divided (where positive) or multiplied by `repetition`; one among
    the answers loses `frequency` for each time and `presence` once.  bias: float32 (N, V) or
    (V,), added.  allowed: int32 (N, ceil(V/32)) or (ceil(V/32),), bit v % 32 of word v / 32 set
    where answer v may be given; the others get -inf, whatever their score.
    out: where the scores go, any of the three types, `scores` or `bias` itself too (default: a new
    float32 tensor)."""
    if _forward_ad._current_level >= 0:
        _no_tangents(scores=scores, repetition=repetition, frequency=frequency, presence=presence, bias=bias, out=out)
    dtype, N, V, device = _rows_of(scores, "scores", _FLOATS)
    T, said, token_stride = 0, None, 0
    if tokens is not None:
        if not (isinstance(tokens, _Tensor) and tokens.dtype is torch.int32 and tokens.get_device() == device
                and tokens.dim() == 2 and tokens.shape[0] == N and (tokens.stride(1) == 1 or tokens.shape[1] < 2)):
            _refuse(tokens, "tokens", (2,), torch.int32, f"({N}, T)", device)
        T, said, token_stride = tokens.shape[1], tokens.data_ptr(), tokens.stride(0)
        lengths = _per_row(lengths, "lengths", torch.int32, N, device)
        prompt = _per_row(prompt, "prompt", torch.int32, N, device)
        repetition = _per_row(repetition, "repetition", torch.float32, N, device)
        frequency = _per_row(frequency, "frequency", torch.float32, N, device)
        presence = _per_row(presence, "presence", torch.float32, N, device)
    elif not (lengths is None and prompt is None and repetition is None and frequency is None and presence is None):
        raise ValueError("lengths, prompt and penalties need tokens.")
    bias, bias_stride = _matrix(bias, "bias", torch.float32, N, V, device)
    allowed, allowed_stride = _matrix(allowed, "allowed", torch.int32, N, (V + 31) // 32, device)
    out, out_type = _result(out, (N, V), device)
    _call(lib.ytm_adjust_scores, device, scores.data_ptr(), dtype, scores.stride(0), N, V, said, token_stride, T,
          lengths, prompt, repetition, frequency, presence, bias, bias_stride, allowed, allowed_stride, out.data_ptr(),
          out_type, out.stride(0))
    return out


def choose(scores: torch.Tensor, temperature: torch.Tensor | None = None, top_k: torch.Tensor | None = None,
           top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
           noise: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One answer for each row of scores (N, V): (index int32 (N,), log probability float32 (N,)).

    temperature (float32 (N,), 0: the best answer), top_k (int32 (N,), 0: no bound), top_p and min_p
    (float32 (N,)) say which answers are kept; the index is that of the largest score / temperature +
    noise of these, the lowest of equal ones, the log probability that of a draw among them.
    noise: float32 (N, V) or (V,), finite; standard Gumbel draws -log(-log(u)) make the answer a
    draw, None the best one.  A row without a score above -inf gets -1 and -inf."""
    if _forward_ad._current_level >= 0:
        _no_tangents(scores=scores, temperature=temperature, top_p=top_p, min_p=min_p, noise=noise)
    dtype, N, V, device = _rows_of(scores, "scores", _FLOATS)
    noise, noise_stride = _matrix(noise, "noise", torch.float32, N, V, device)
    temperature = _per_row(temperature, "temperature", torch.float32, N, device)
    top_k = _per_row(top_k, "top_k", torch.int32, N, device)
    top_p = _per_row(top_p, "top_p", torch.float32, N, device)
    min_p = _per_row(min_p, "min_p", torch.float32, N, device)
    where = scores.device
    tokens = torch.empty(N, dtype=torch.int32, device=where)
    logprobs = torch.empty(N, dtype=torch.float32, device=where)
    need, workspace = 0, None
    if V >= 32768 and N <= 64:  # fewer or more rows are not sliced
        need, workspace = _workspace(lib.ytm_choose_workspace, where, dtype, N, V)
    _call(lib.ytm_choose, device, scores.data_ptr(), dtype, scores.stride(0), N, V, temperature, top_k, top_p, min_p,
          noise, noise_stride, tokens.data_ptr(), logprobs.data_ptr(), workspace.data_ptr() if need else None, need)
    return tokens, logprobs
