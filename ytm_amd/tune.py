"""Adapting a model's answers and learning from them, on the GPU (not in the reference).

A model whose weights are held in 4 bits (ytm_amd.decode) serves many users, each with low-rank corrections
of its own, which learn from the answers that were given:

    adapters = tune.Adapters(count=64, clauses=C, outputs=K, rank=16)
    scores = decode.readout(bits, codes, scales, clauses=C)          # class sums (N, K)
    hidden = adapters.adapt(scores, bits, which)                     # in place, a user's adapter a row
    token, logprob = decode.choose(scores, temperature=t, noise=...)
    # ... what the answers were worth comes back: advantages; or which of two answers was preferred
    losses, grad, _ = tune.policy_loss(scores, token, logprob, advantages, temperature=t)
    adapters.learn(grad, bits, which, hidden, lr=1e-3)

The operators take torch tensors on one GPU and put their work on the current stream of that GPU without
waiting for it (they may be captured into a graph, Adapters and AdamW made before).  Rows may be any distance
apart; a row's elements follow one another.  A wrong argument raises TypeError or ValueError before anything is
launched.  Gradients are explicit: a loss returns the scores' gradient, adapt_gradient takes any gradient of
adapt's output, and nothing is recorded by autograd, so tensors that require a gradient, or have a tangent
of forward mode, are refused.  The formulas are at ytm_adapt, ytm_adapt_gradient, ytm_policy_loss,
ytm_preference_loss and ytm_adamw in include/ytm.h.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad as _forward_ad

from ._lib import DTYPE_BITS, AdamWTensor, check, lib
from .decode import (_call, _changed, _CLAUSES, _FLOATS, _no_tangents, _per_row, _refuse, _result, _rows_of, _Tensor)

_BLOCK = 256  # elements of a state in 8 bits that share a scale


def _adapters(t, name: str, dtype: torch.dtype | None, shape: tuple | None, device: int) -> tuple[int, int]:
    """(distance from an adapter to the next, from a row to the next) of adapters (M, rows, width); any where
    `dtype` or `shape` is None."""
    if isinstance(t, _Tensor) and t.get_device() == device and t.dim() == 3 and not t.requires_grad:
        per_adapter, per_row, one = t.stride()
        adapters, rows, width = size = t.shape
        if ((size == shape or shape is None) and (t.dtype is dtype or dtype is None and t.dtype in _FLOATS)
                and (one == 1 or width < 2)):
            return (per_adapter if adapters > 1 else 0), (per_row if rows > 1 else 0)
    fits = shape is None or isinstance(t, _Tensor) and tuple(t.shape) == shape
    _refuse(t, name, (3,), _FLOATS if dtype is None else dtype, "" if fits else str(shape), device)
    return (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else 0)


def _clauses(x, C: int, rows: int, device: int) -> int:
    """The type code of clause outputs x (rows, C)."""
    width = -(-C // 32) if isinstance(x, _Tensor) and x.dtype is torch.int32 else C
    if not (isinstance(x, _Tensor) and x.get_device() == device and x.dtype in _CLAUSES and x.shape == (rows, width)
            and (x.stride(1) == 1 or width < 2) and not x.requires_grad):
        fits = isinstance(x, _Tensor) and tuple(x.shape) == (rows, width)
        _refuse(x, "x", (2,), _CLAUSES, "" if fits else f"({rows}, {width})", device)
    return _CLAUSES[x.dtype]


@functools.lru_cache(maxsize=4096)
def _bytes(name: str, *args: int) -> int:
    """What the library's `name` says that a workspace takes."""
    need = ctypes.c_int64()
    check(getattr(lib, name)(*args, need))
    return need.value


def _hidden(t, rows: int, rank: int, device: int) -> None:
    if not (isinstance(t, _Tensor) and t.dtype is torch.float32 and t.get_device() == device and t.shape == (rows, rank)
            and (t.stride(1) == 1 or rank < 2) and not t.requires_grad):
        fits = isinstance(t, _Tensor) and tuple(t.shape) == (rows, rank)
        _refuse(t, "hidden", (2,), torch.float32, "" if fits else f"({rows}, {rank})", device)


def _number(v, name: str) -> float:
    v = float(v)
    if not math.isfinite(v):
        raise ValueError(f"{name} must be finite.")
    return v


def adapt(scores: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, which: torch.Tensor,
          scale: float = 1.0, hidden: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Scores (N, K) with each row's low-rank correction: scores[n] + scale * up[a] (down[a] x[n]), a = which[n].

    x: the clause outputs that readout made the scores of: bits, int32 (N, ceil(C/32)), or float32, float16 or
    bfloat16 (N, C).  down (M, r, C) and up (M, K, r): the adapters, float32, float16 or bfloat16, r up to 256.
    which: int32 (N,), each row's adapter; a row whose number is outside 0..M-1 keeps its scores.
    hidden: where down[a] x[n] goes, float32 (N, r), for adapt_gradient.  out: where the scores go, any of the
    three types, `scores` itself too (default: a new float32 tensor)."""
    if _forward_ad._current_level >= 0:
        _no_tangents(scores=scores, x=x, down=down, up=up, hidden=hidden, out=out)
    scale = _number(scale, "scale")
    dtype, N, K, device = _rows_of(scores, "scores", _FLOATS)
    down_adapter, down_rank = _adapters(down, "down", None, None, device)
    M, r, C = down.shape
    up_adapter, up_output = _adapters(up, "up", down.dtype, (M, K, r), device)
    x_type = _clauses(x, C, N, device)
    which = _per_row(which, "which", torch.int32, N, device)
    if which is None:
        raise TypeError("which must be a torch tensor.")
    if hidden is not None:
        _hidden(hidden, N, r, device)
        _changed((hidden,))
    out, out_type = _result(out, (N, K), device)
    need = _bytes("ytm_adapt_workspace", N, C, M, r)
    workspace = torch.empty(need, dtype=torch.uint8, device=scores.device) if need else None
    _call(lib.ytm_adapt, device, scores.data_ptr(), dtype, scores.stride(0), N, K, x.data_ptr(), x_type, x.stride(0), C,
          down.data_ptr(), down_adapter, down_rank, up.data_ptr(), up_adapter, up_output, _FLOATS[down.dtype], M, r,
          which, scale, None if hidden is None else hidden.data_ptr(), 0 if hidden is None else hidden.stride(0),
          out.data_ptr(), out_type, out.stride(0), workspace.data_ptr() if need else None, need)
    return out


def adapt_gradient(grad: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, which: torch.Tensor,
                   hidden: torch.Tensor, scale: float = 1.0,
                   out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The gradients (M, r, C) of down and (M, K, r) of up, where grad (N, K) is that of adapt's output and
    hidden what adapt gave; the other operands are adapt's.  Adapters that no row names get 0.  The gradient
    of adapt's scores is grad itself; clause outputs have none.
    out: where the two go, both of the adapters' type (default: new tensors) or both float32, for sums below what
    float16 holds."""
    if _forward_ad._current_level >= 0:
        _no_tangents(grad=grad, x=x, up=up, hidden=hidden)
        if out is not None:
            _no_tangents(down_gradient=out[0], up_gradient=out[1])
    scale = _number(scale, "scale")
    dtype, N, K, device = _rows_of(grad, "grad", _FLOATS)
    _adapters(down, "down", None, None, device)
    M, r, C = down.shape
    w = down.dtype
    up_adapter, up_output = _adapters(up, "up", w, (M, K, r), device)
    x_type = _clauses(x, C, N, device)
    which = _per_row(which, "which", torch.int32, N, device)
    if which is None:
        raise TypeError("which must be a torch tensor.")
    _hidden(hidden, N, r, device)
    if out is None:
        out = torch.empty((M, r, C), dtype=w, device=grad.device), torch.empty((M, K, r), dtype=w, device=grad.device)
    d_down, d_up = out
    kind = torch.float32 if isinstance(d_down, _Tensor) and d_down.dtype is torch.float32 else w
    d_down_adapter, d_down_rank = _adapters(d_down, "out[0]", kind, (M, r, C), device)
    d_up_adapter, d_up_output = _adapters(d_up, "out[1]", kind, (M, K, r), device)
    _changed((d_down, d_up))
    need = _bytes("ytm_adapt_gradient_workspace", N, C, K, M, r)
    workspace = torch.empty(need, dtype=torch.uint8, device=grad.device) if need else None
    _call(lib.ytm_adapt_gradient_as, device, grad.data_ptr(), dtype, grad.stride(0), N, K, x.data_ptr(), x_type,
          x.stride(0), C, up.data_ptr(), up_adapter, up_output, _FLOATS[w], M, r, which, scale, hidden.data_ptr(),
          hidden.stride(0), _FLOATS[kind], d_down.data_ptr(), d_down_adapter, d_down_rank, d_up.data_ptr(), d_up_adapter,
          d_up_output, workspace.data_ptr() if need else None, need)
    return d_down, d_up


def policy_loss(scores: torch.Tensor, tokens: torch.Tensor, old: torch.Tensor, advantages: torch.Tensor,
                reference: torch.Tensor | None = None, kl: float = 0.0, clip: float = 0.2,
                clip_high: float | None = None, weights: torch.Tensor | None = None,
                temperature: torch.Tensor | None = None, out: torch.Tensor | None = None
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Clipped policy loss of drawn answers: (losses (N,), the gradient of their sum by scores (N, V), log
    probabilities (N,)).

    tokens: int32 (N,), the answers; a row whose answer is outside 0..V-1 (-1) or has a score of -inf is left
    out.  old: float32 (N,), their log probabilities when they were drawn, as choose gives them (without
    filters).  advantages: float32 (N,), what they were worth.  The ratio of the probabilities counts up
    to 1 + clip_high (default: clip) and down to 1 - clip.  reference: float32 (N,), their log probabilities by
    the model that kl draws the answers towards.  weights: float32 (N,), each row's (default 1 / N; a row of 0,
    such as one that fills a batch, has a loss and gradient of 0 whatever its other numbers).  temperature:
    float32 (N,), as for choose.
    out: where the gradient goes, any of the three types, `scores` itself too (default: a new float32 tensor)."""
    if _forward_ad._current_level >= 0:
        _no_tangents(scores=scores, old=old, advantages=advantages, reference=reference, weights=weights,
                     temperature=temperature, out=out)
    dtype, N, V, device = _rows_of(scores, "scores", _FLOATS)
    if tokens is None or old is None or advantages is None:
        raise TypeError("tokens, old and advantages must be torch tensors.")
    tokens = _per_row(tokens, "tokens", torch.int32, N, device)
    old = _per_row(old, "old", torch.float32, N, device)
    advantages = _per_row(advantages, "advantages", torch.float32, N, device)
    reference = _per_row(reference, "reference", torch.float32, N, device)
    weights = _per_row(weights, "weights", torch.float32, N, device)
    temperature = _per_row(temperature, "temperature", torch.float32, N, device)
    kl, clip = _number(kl, "kl"), _number(clip, "clip")
    clip_high = clip if clip_high is None else _number(clip_high, "clip_high")
    if kl and reference is None:
        raise ValueError("kl needs a reference.")
    out, out_type = _result(out, (N, V), device)
    where = scores.device
    losses, logprobs = (torch.empty(N, dtype=torch.float32, device=where) for _ in range(2))
    need = _bytes("ytm_policy_loss_workspace", N, V)
    workspace = torch.empty(need, dtype=torch.uint8, device=where) if need else None
    _call(lib.ytm_policy_loss, device, scores.data_ptr(), dtype, scores.stride(0), N, V, tokens, old, advantages,
          reference, kl, clip, clip_high, weights, temperature, losses.data_ptr(),
          logprobs.data_ptr(), out.data_ptr(), out_type, out.stride(0), workspace.data_ptr() if need else None, need)
    return losses, out, logprobs


def preference_loss(scores: torch.Tensor, tokens: torch.Tensor, starts: torch.Tensor, reference: torch.Tensor,
                    beta: float = 0.1, smoothing: float = 0.0, temperature: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Loss of answers of which one of two was preferred: (losses (P,), the gradient of their sum by scores
    (N, V), log probabilities of the sequences (2 P,)).

    Rows starts[s] .. starts[s + 1] - 1 (int32 (2 P + 1,), not falling) are sequence s; of pair p sequence 2 p is the
    preferred one, 2 p + 1 the other.  tokens: int32 (N,), each row's answer (-1: none).  reference: float32
    (2 P,), the sequences' log probabilities by the model that the learning begins with.  beta: how far from
    it they may go.  smoothing: the chance that a preference is the wrong way round.  temperature: float32
    (N,), as for choose.  Rows of no sequence get a gradient of 0.
    out: where the gradient goes, any of the three types, `scores` itself too (default: a new float32 tensor)."""
    if _forward_ad._current_level >= 0:
        _no_tangents(scores=scores, reference=reference, temperature=temperature, out=out)
    dtype, N, V, device = _rows_of(scores, "scores", _FLOATS)
    if tokens is None or starts is None or reference is None:
        raise TypeError("tokens, starts and reference must be torch tensors.")
    tokens = _per_row(tokens, "tokens", torch.int32, N, device)
    pairs = starts.shape[0] // 2 if isinstance(starts, _Tensor) and starts.dim() == 1 else 0
    if pairs < 1:
        _refuse(starts, "starts", (1,), torch.int32, "(2 P + 1,)", device)
    starts = _per_row(starts, "starts", torch.int32, 2 * pairs + 1, device)
    reference = _per_row(reference, "reference", torch.float32, 2 * pairs, device)
    temperature = _per_row(temperature, "temperature", torch.float32, N, device)
    beta, smoothing = _number(beta, "beta"), _number(smoothing, "smoothing")
    out, out_type = _result(out, (N, V), device)
    where = scores.device
    losses, logprobs = (torch.empty(n, dtype=torch.float32, device=where) for n in (pairs, 2 * pairs))
    need = _bytes("ytm_preference_loss_workspace", N, V)
    workspace = torch.empty(need, dtype=torch.uint8, device=where) if need else None
    _call(lib.ytm_preference_loss, device, scores.data_ptr(), dtype, scores.stride(0), N, V, tokens, starts, pairs,
          reference, beta, smoothing, temperature, losses.data_ptr(), logprobs.data_ptr(), out.data_ptr(), out_type,
          out.stride(0), workspace.data_ptr() if need else None, need)
    return losses, out, logprobs


class AdamW:
    """AdamW over many tensors at once, with states in 32 or in 8 bits.

    parameters: float32, float16 or bfloat16; gradients: one for each, of the same shape, of the same type or
    float32.  Both are contiguous tensors on one GPU that stay where they are: a step reads and writes them in
    place.  The states are lists of tensors of the parameters' shapes: first (the mean of the gradients) and
    second (that of their squares), float32; with bits=8 float8_e4m3fn, times first_scales and second_scales,
    float32 powers of two for each 256 elements in a row, and second is held as its root.  steps: int64, the
    steps that each tensor has made.

    Sums and states are float32 while a step is made (with bits=8 m / (sqrt(v) + eps) to two units in its last
    place).  What is stored in fewer bits, 16-bit parameters too, is rounded up or down at random with the chances
    that keep its mean, the same ones for the same `seed`: an average that moves by a thousandth a step would
    never leave an 8-bit number's neighbourhood otherwise.

    states: first, second (and the scales) to go on with, as `states()` gives them, and steps the number of
    steps made, a number or a tensor of one for each parameter; by default all begin at 0.

    A copy (copy.deepcopy, pickle, torch.save) steps the copied tensors, a shallow one the same as its original."""

    def __init__(self, parameters: list[torch.Tensor], gradients: list[torch.Tensor], bits: int = 32,
                 states: dict[str, list[torch.Tensor]] | None = None, steps: int | torch.Tensor = 0, seed: int = 0):
        if bits not in (8, 32):
            raise ValueError("bits must be 8 or 32.")
        self.bits, self.seed = int(bits), int(seed) & 0xFFFFFFFF
        self.parameters, self.gradients = list(parameters), list(gradients)
        if not self.parameters:
            raise ValueError("there are no parameters.")
        if len(self.gradients) != len(self.parameters):
            raise ValueError(f"there are {len(self.parameters)} parameters and {len(self.gradients)} gradients.")
        first = self.parameters[0]
        self._device = first.get_device() if isinstance(first, _Tensor) else -1
        for i, (p, g) in enumerate(zip(self.parameters, self.gradients)):
            self._whole(p, f"parameters[{i}]", _FLOATS, None)
            self._whole(g, f"gradients[{i}]", (p.dtype, torch.float32), p.shape)
            if g.requires_grad:
                raise ValueError(f"gradients[{i}] requires a gradient; this operator has none.")
        names = ["first", "second"] + (["first_scales", "second_scales"] if bits == 8 else [])
        if states is not None and sorted(states) != sorted(names):
            raise ValueError(f"states must hold {', '.join(names)}.")
        for name in names:
            scales = name.endswith("scales")
            dtype = torch.float32 if bits == 32 or scales else torch.float8_e4m3fn
            shapes = [torch.Size((-(-p.numel() // _BLOCK),)) if scales else p.shape for p in self.parameters]
            if states is None:
                held = [torch.zeros(s, dtype=dtype, device=first.device) for s in shapes]
            else:
                held = list(states[name])
                if len(held) != len(shapes):
                    raise ValueError(f"states[{name!r}] must hold {len(shapes)} tensors, not {len(held)}.")
                for i, (t, s) in enumerate(zip(held, shapes)):
                    self._whole(t, f"{name}[{i}]", (dtype,), s)
            setattr(self, name, held)
        if isinstance(steps, _Tensor):
            if steps.shape != (len(self.parameters),) or steps.is_floating_point():
                raise ValueError(f"steps must be whole numbers of shape ({len(self.parameters)},).")
            if bool((steps < 0).any()):
                raise ValueError("steps must be 0 or more.")
            self._steps = steps.detach().to(device=first.device, dtype=torch.int64, copy=True).contiguous()
        else:
            if steps < 0:
                raise ValueError("steps must be 0 or more.")
            self._steps = torch.full((len(self.parameters),), int(steps), dtype=torch.int64, device=first.device)
        self._names = names
        self._written = tuple(t for name in ("parameters", *names) for t in getattr(self, name))
        self._apart()
        self._make_table()

    def _whole(self, t, name: str, dtypes, shape) -> None:
        if not isinstance(t, _Tensor):
            raise TypeError(f"{name} must be a torch tensor.")
        if not t.is_cuda:
            raise ValueError(f"{name} must be on a GPU.")
        if t.get_device() != self._device:
            raise ValueError(f"{name} must be on cuda:{self._device}, not {t.device}.")
        if t.dtype not in dtypes:
            names = " or ".join(str(d).removeprefix("torch.") for d in dict.fromkeys(dtypes))
            raise TypeError(f"{name} must be {names}, not {t.dtype}.")
        if shape is not None and t.shape != shape:
            raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}.")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous.")
        if _forward_ad._current_level >= 0:
            _no_tangents(**{name: t})

    def _apart(self) -> None:
        """What is written must not share memory with anything else."""
        spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), True) for t in self._written if t.numel()]
        spans += [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), False) for t in self.gradients if t.numel()]
        written_to = read_to = 0
        for begin, end, written in sorted(spans):
            if begin < written_to or written and begin < read_to:
                raise ValueError("parameters and states must not overlap each other or the gradients.")
            if written:
                written_to = max(written_to, end)
            else:
                read_to = max(read_to, end)

    def _make_table(self) -> None:
        n = len(self.parameters)
        rows = (AdamWTensor * n)()
        for i, row in enumerate(rows):
            p, g = self.parameters[i], self.gradients[i]
            row.parameter, row.gradient, row.count = p.data_ptr(), g.data_ptr(), p.numel()
            row.parameter_dtype, row.gradient_dtype = _FLOATS[p.dtype], _FLOATS[g.dtype]
            for name in self._names:
                setattr(row, name, getattr(self, name)[i].data_ptr())
        size, self._chunks, self._count = ctypes.c_int64(), ctypes.c_int64(), n
        check(lib.ytm_adamw_table(rows, n, self.bits, None, size, self._chunks))
        host = torch.empty(size.value, dtype=torch.uint8, device="cpu")  # whatever torch's default is
        check(lib.ytm_adamw_table(rows, n, self.bits, host.data_ptr(), size, self._chunks))
        self._table = host.to(self.parameters[0].device)
        # the memory that the table's addresses mean
        self._held = [t.detach() for t in (*self._written, *self.gradients)]

    def __getstate__(self) -> dict:
        # the table's addresses are those of this object's tensors; pickle alone does not know float8
        state = {k: v for k, v in self.__dict__.items() if k not in ("_table", "_chunks", "_held", "_written")}
        if self.bits == 8:
            state |= {name: [t.view(torch.uint8) for t in state[name]] for name in ("first", "second")}
        return state

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        if self.bits == 8:
            self.first, self.second = ([t.view(torch.float8_e4m3fn) for t in s] for s in (self.first, self.second))
        AdamW.__init__(self, self.parameters, self.gradients, self.bits, self.states(), self.steps, self.seed)
        self._steps = state["_steps"]

    @property
    def steps(self) -> torch.Tensor:
        return self._steps

    @steps.setter
    def steps(self, steps: torch.Tensor) -> None:
        if _per_row(steps, "steps", torch.int64, self._count, self._device) is None:
            raise TypeError("steps must be a torch tensor.")
        self._steps = steps

    def states(self) -> dict[str, list[torch.Tensor]]:
        """The states, to go on with: AdamW(..., states=a.states(), steps=a.steps)."""
        return {name: getattr(self, name) for name in self._names}

    def step(self, lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
             weight_decay: float = 0.01, active: torch.Tensor | None = None) -> None:
        """One step of all tensors: the states take in the gradients, the parameters move.

        lr: a number, or a float32 tensor () on the GPU, which a captured graph reads again at each replay.
        active: bool, one for each tensor, on the GPU; the tensors for which it is false stay as they are."""
        n, rate_at, flags = self._count, None, None  # as many as the table has
        if isinstance(lr, _Tensor):
            if lr.dtype is not torch.float32 or lr.numel() != 1 or lr.get_device() != self._device:
                raise ValueError(f"lr must be a number or one float32 on cuda:{self._device}.")
            rate_at, lr = lr.data_ptr(), 0.0
        if active is not None:
            flags = _per_row(active, "active", torch.bool, n, self._device)
        _changed(self._written)
        _call(lib.ytm_adamw, self._device, self._table.data_ptr(), n, self._chunks.value, self.bits,
              self._steps.data_ptr(), flags, _number(lr, "lr"), rate_at, float(betas[0]), float(betas[1]), _number(eps, "eps"),
              _number(weight_decay, "weight_decay"), self.seed)


class Adapters:
    """Low-rank adapters of many users beside one model's readout, and what they learn with.

    down (count, rank, clauses) starts as small random numbers, up (count, outputs, rank) as 0, so that nothing
    changes before something is learnt.  gradients: those of the last learn(), float32 where the adapters are
    float16, which holds nothing below 6e-8: means over a batch of unlikely answers are less.  optimizer: an AdamW
    whose tensors are down[a] and up[a] of each adapter a, in turn, with states of `bits` bits.  down, up and
    gradients stay where they are: what is to be in them is copied into them.  A copy of the whole (copy.deepcopy,
    pickle, torch.save) has adapters, states and step counts of its own."""

    def __init__(self, count: int, clauses: int, outputs: int, rank: int = 16, scale: float = 1.0,
                 dtype: torch.dtype = torch.float32, bits: int = 32, device: str | torch.device = "cuda", seed: int = 0):
        if min(count, clauses, outputs, rank) < 1:
            raise ValueError("count, clauses, outputs and rank must be positive.")
        if rank > 256:
            raise ValueError("rank must be at most 256.")
        if dtype not in _FLOATS:
            raise TypeError("adapters are float32, float16 or bfloat16.")
        g = torch.Generator(device=device).manual_seed(int(seed))
        self.count, self.scale = int(count), _number(scale, "scale")
        down = torch.empty(count, rank, clauses, dtype=torch.float32, device=device)
        self.down = down.normal_(0.0, clauses ** -0.5, generator=g).to(dtype)
        self.up = torch.zeros(count, outputs, rank, dtype=dtype, device=device)
        kind = torch.float32 if dtype is torch.float16 else dtype
        self.gradients = torch.zeros_like(self.down, dtype=kind), torch.zeros_like(self.up, dtype=kind)
        self.optimizer = AdamW(*self._each(), bits=bits, seed=seed)

    def _each(self) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
        each = lambda down, up: [t for a in range(self.count) for t in (down[a], up[a])]  # noqa: E731
        return each(self.down, self.up), each(*self.gradients)

    def __getstate__(self) -> dict:
        # the optimiser's parameters and gradients are parts of this object's tensors, which pickle would part
        optimizer = self.optimizer.__getstate__()
        del optimizer["parameters"], optimizer["gradients"]
        return dict(self.__dict__, optimizer=optimizer)

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        parameters, gradients = self._each()
        self.optimizer = AdamW.__new__(AdamW)
        self.optimizer.__setstate__(dict(state["optimizer"], parameters=parameters, gradients=gradients))

    def adapt(self, scores: torch.Tensor, x: torch.Tensor, which: torch.Tensor) -> torch.Tensor:
        """Corrects scores (N, K) in place, each row by its adapter, and returns what learn() needs (N, rank)."""
        rows = which.shape[0] if isinstance(which, _Tensor) and which.dim() == 1 else 0  # adapt says what is wrong
        hidden = torch.empty(rows, self.down.shape[1], dtype=torch.float32, device=self.down.device)
        adapt(scores, x, self.down, self.up, which, self.scale, hidden=hidden, out=scores)
        return hidden

    def learn(self, grad: torch.Tensor, x: torch.Tensor, which: torch.Tensor, hidden: torch.Tensor,
              lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
              weight_decay: float = 0.01) -> None:
        """A step of the adapters that `which` names, by the gradient (N, K) of the scores that adapt() made."""
        o = self.optimizer
        if [t.data_ptr() for t in (self.down, self.up, *self.gradients)] != [
                t.data_ptr() for t in (*o.parameters[:2], *o.gradients[:2])]:
            raise ValueError("down, up and gradients must be the tensors that the optimizer steps; copy into them.")
        adapt_gradient(grad, x, self.down, self.up, which, hidden, self.scale, out=self.gradients)
        # rows without an adapter, -1 and count, mark what is after the last
        named = torch.zeros(self.count + 1, 2, dtype=torch.bool, device=which.device)
        named.index_fill_(0, which.clamp(-1, self.count).long(), True)
        o.step(lr, betas, eps, weight_decay, active=named.view(-1)[:-2])
