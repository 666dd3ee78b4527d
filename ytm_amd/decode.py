"""From clause outputs to an answer, on the GPU (not in the reference).

A model with many outputs, such as one a word of a vocabulary, answers in three steps:

    codes, scales = decode.pack_weights(tm.get_weights())          # once: weights in 4 bits
    bits = decode.pack_outputs(tm.transform(X))                    # clause outputs, packed
    scores = decode.readout(bits, codes, scales, clauses=C)        # class sums (N, K)
    scores = decode.adjust_scores(scores, tokens=said, ...)        # penalties, bias, grammar
    token, logprob = decode.choose(scores, top_p=..., noise=...)   # the answer of each row

readout, adjust_scores and choose take torch tensors on one GPU and put their work on the
current stream of that GPU without waiting for it, as torch's own operations do (they may be
captured into a graph); pack_weights and pack_outputs turn the framework's host arrays into such
tensors.  Rows may be any distance apart; a row's elements follow one another.  A wrong argument
raises TypeError or ValueError before anything is launched.  There are no gradients: clause
outputs are bits made by automata and the codes are made from trained weights, so tensors that
require a gradient are refused.  The formulas are at ytm_readout, ytm_adjust_scores and ytm_choose
in include/ytm.h.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from ._lib import DTYPE_BF16, DTYPE_BITS, DTYPE_F16, DTYPE_F32, check, lib

_FLOATS = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}
# E2M1 magnitudes of the codes 0..7, and the points between them
_MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], np.float32)
_BETWEEN = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])


def pack_weights(weights: np.ndarray, group: int = 32, dtype: torch.dtype = torch.float32,
                 device: str | torch.device = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """Clause weights (C, K), as get_weights() gives them, in 4 bits for readout: codes uint8
    (K, 16 ceil(C/32)) and scales (K, ceil(C/group)) of `dtype`.  A group's largest weight becomes
    6 (a code's largest value) times its scale, the others the nearest code, ties to the smaller
    magnitude.  Runs on the host."""
    w = np.asarray(weights, dtype=np.float32)
    if w.ndim != 2:
        raise ValueError("weights must have shape (clauses, outputs).")
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
    # a scale that its type holds as 0 or infinity has no codes; 1 leaves zeros as they are
    scales = torch.where((scales > 0) & torch.isfinite(scales), scales, torch.ones((), dtype=dtype))
    per_clause = scales.double().numpy().repeat(group, axis=1)[:, :C]
    scaled = w.T / per_clause  # in float64, so that the nearest code is
    code = np.zeros((K, padded), np.uint8)
    code[:, :C] = np.searchsorted(_BETWEEN, np.abs(scaled), side="left") | (scaled < 0).astype(np.uint8) << 3
    return torch.from_numpy(code[:, 0::2] | code[:, 1::2] << 4).to(device), scales.to(device)


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


def _operand(t, name: str, dims, device=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor.")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} must be on {'a GPU' if device is None else device}.")
    if t.dim() not in dims:
        raise ValueError(f"{name} must have {' or '.join(map(str, dims))} dimensions.")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient; this operator has none.")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}'s rows must be contiguous.")
    return t


def _float_type(t: torch.Tensor, name: str) -> int:
    code = _FLOATS.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}.")
    return code


def _matrix(t, name: str, dtype: torch.dtype, rows: int, width: int, device) -> tuple[int | None, int]:
    """(address, row stride; 0 for one row shared by all) of an optional operand (rows, width) or
    (width)."""
    if t is None:
        return None, 0
    _operand(t, name, (1, 2), device)
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}.")
    if t.shape[-1] != width or (t.dim() == 2 and t.shape[0] != rows):
        raise ValueError(f"{name} must have shape ({rows}, {width}) or ({width},), not {tuple(t.shape)}.")
    return t.data_ptr(), t.stride(0) if t.dim() == 2 and rows > 1 else 0


def _per_row(t, name: str, dtype: torch.dtype, rows: int, device) -> int | None:
    if t is None:
        return None
    _operand(t, name, (1,), device)
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}.")
    if t.shape[0] != rows:
        raise ValueError(f"{name} must have {rows} elements, not {t.shape[0]}.")
    return t.data_ptr()


def _result(out, name: str, shape: tuple[int, int], device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.float32, device=device)
    _operand(out, name, (2,), device)
    if tuple(out.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(out.shape)}.")
    return out


def _call(function, device: torch.device, *args) -> None:
    """function(*args, current stream) with `device` current."""
    if device.index == torch.cuda.current_device():
        check(function(*args, torch.cuda.current_stream(device).cuda_stream))
    else:
        with torch.cuda.device(device):
            check(function(*args, torch.cuda.current_stream(device).cuda_stream))


def readout(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, group: int = 32, clauses: int | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """Class sums (N, K) of clause outputs x through weights in 4 bits (pack_weights).

    x: bits, int32 (N, ceil(C/32)) as pack_outputs gives them, C being `clauses` (default: every
    bit); or float32, float16 or bfloat16 (N, C), outputs averaged over models or patches.
    out: where the sums go, float32, float16 or bfloat16 (default: a new float32 tensor)."""
    _operand(x, "x", (2,))
    device = x.device
    N, width = x.shape
    if x.dtype == torch.int32:
        x_type = DTYPE_BITS
        C = 32 * width if clauses is None else int(clauses)
        if not -(-C // 32) == width:
            raise ValueError(f"x must hold {-(-C // 32)} words of clause bits a row, not {width}.")
    else:
        x_type = _float_type(x, "x")
        C = width
        if clauses is not None and int(clauses) != C:
            raise ValueError(f"x must have {clauses} columns, not {C}.")
    _operand(codes, "codes", (2,), device)
    _operand(scales, "scales", (2,), device)
    if codes.dtype != torch.uint8:
        raise TypeError("codes must be uint8.")
    K, group = codes.shape[0], int(group)
    if group < 32 or group % 32:
        raise ValueError("group must be a multiple of 32.")
    if codes.shape[1] < 16 * -(-C // 32):
        raise ValueError(f"codes must hold {16 * -(-C // 32)} bytes an output, not {codes.shape[1]}.")
    if scales.shape[0] != K or scales.shape[1] != -(-C // group):
        raise ValueError(f"scales must have shape ({K}, {-(-C // group)}), not {tuple(scales.shape)}.")
    scale_type = _float_type(scales, "scales")
    out = _result(out, "out", (N, K), device)
    out_type = _float_type(out, "out")
    need = ctypes.c_int64()
    check(lib.ytm_readout_workspace(x_type, N, C, K, ctypes.byref(need)))
    workspace = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
    _call(lib.ytm_readout, device, x.data_ptr(), x_type, x.stride(0), N, C, codes.data_ptr(), codes.stride(0),
          scales.data_ptr(), scale_type, scales.stride(0), group, K, out.data_ptr(), out_type, out.stride(0),
          None if workspace is None else workspace.data_ptr(), need.value)
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
    out: where the scores go, any of the three types, `scores` itself too (default: a new float32
    tensor)."""
    _operand(scores, "scores", (2,))
    device = scores.device
    N, V = scores.shape
    dtype = _float_type(scores, "scores")
    T, said, token_stride = 0, None, 0
    if tokens is not None:
        _operand(tokens, "tokens", (2,), device)
        if tokens.dtype != torch.int32:
            raise TypeError("tokens must be int32.")
        if tokens.shape[0] != N:
            raise ValueError(f"tokens must have {N} rows, not {tokens.shape[0]}.")
        T, said, token_stride = tokens.shape[1], tokens.data_ptr(), tokens.stride(0)
    elif not (lengths is None and prompt is None and repetition is None and frequency is None and presence is None):
        raise ValueError("lengths, prompt and penalties need tokens.")
    bias_at, bias_stride = _matrix(bias, "bias", torch.float32, N, V, device)
    allowed_at, allowed_stride = _matrix(allowed, "allowed", torch.int32, N, -(-V // 32), device)
    out = _result(out, "out", (N, V), device)
    _call(lib.ytm_adjust_scores, device, scores.data_ptr(), dtype, scores.stride(0), N, V, said, token_stride, T,
          _per_row(lengths, "lengths", torch.int32, N, device), _per_row(prompt, "prompt", torch.int32, N, device),
          _per_row(repetition, "repetition", torch.float32, N, device),
          _per_row(frequency, "frequency", torch.float32, N, device),
          _per_row(presence, "presence", torch.float32, N, device), bias_at, bias_stride, allowed_at, allowed_stride,
          out.data_ptr(), _float_type(out, "out"), out.stride(0))
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
    _operand(scores, "scores", (2,))
    device = scores.device
    N, V = scores.shape
    dtype = _float_type(scores, "scores")
    noise_at, noise_stride = _matrix(noise, "noise", torch.float32, N, V, device)
    tokens = torch.empty(N, dtype=torch.int32, device=device)
    logprobs = torch.empty(N, dtype=torch.float32, device=device)
    _call(lib.ytm_choose, device, scores.data_ptr(), dtype, scores.stride(0), N, V,
          _per_row(temperature, "temperature", torch.float32, N, device),
          _per_row(top_k, "top_k", torch.int32, N, device), _per_row(top_p, "top_p", torch.float32, N, device),
          _per_row(min_p, "min_p", torch.float32, N, device), noise_at, noise_stride, tokens.data_ptr(),
          logprobs.data_ptr())
    return tokens, logprobs
