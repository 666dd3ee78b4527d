"""What the answering operators refuse of their operands, before anything is launched.

Tensors here are on the CPU and say that they are on a GPU; the library's entries only count their
calls, so a call that is let through is seen and reads nothing.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as forward_ad  # noqa: E402

from ytm_amd import _lib, decode  # noqa: E402


class OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def on_gpu(*shape, dtype=torch.float32, grad=False):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu).requires_grad_(grad)


class Entries:
    """The library's entries: how often one that launches was called."""

    launched = 0

    def __getattr__(self, name):
        def entry(*args):
            self.launched += not name.endswith("_workspace")
            return 0

        return entry


@pytest.fixture
def entries(monkeypatch):
    e = Entries()
    monkeypatch.setattr(decode, "lib", e)
    monkeypatch.setattr(decode, "_device_now", lambda: 0)
    monkeypatch.setattr(decode, "_stream_of", lambda device: 0)
    return e


def readout(**kw):
    a = dict(x=on_gpu(2, 64), codes=on_gpu(3, 32, dtype=torch.uint8), scales=on_gpu(3, 2), out=on_gpu(2, 3))
    return decode.readout(**{**a, **kw})


def adjust(**kw):
    a = dict(scores=on_gpu(2, 10), tokens=on_gpu(2, 4, dtype=torch.int32), out=on_gpu(2, 10))
    return decode.adjust_scores(**{**a, **kw})


def choose(**kw):
    return decode.choose(**{**dict(scores=on_gpu(2, 10)), **kw})


FLOATS = [
    (readout, "x", (2, 64)), (readout, "scales", (3, 2)), (readout, "out", (2, 3)),
    (adjust, "scores", (2, 10)), (adjust, "repetition", (2,)), (adjust, "frequency", (2,)),
    (adjust, "presence", (2,)), (adjust, "bias", (2, 10)), (adjust, "bias", (10,)), (adjust, "out", (2, 10)),
    (choose, "scores", (2, 10)), (choose, "temperature", (2,)), (choose, "top_p", (2,)), (choose, "min_p", (2,)),
    (choose, "noise", (2, 10)), (choose, "noise", (10,)),
]


@pytest.mark.parametrize("call,name,shape", FLOATS)
def test_operands_that_require_a_gradient(entries, call, name, shape):
    """Refused where gradients are recorded, taken where none are: what a trained module's parameters are."""
    with pytest.raises(ValueError, match="gradient"):
        call(**{name: on_gpu(*shape, grad=True)})
    assert entries.launched == 0
    with torch.no_grad():
        call(**{name: on_gpu(*shape, grad=True)})
    assert entries.launched == 1


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call,name,shape", [
    (readout, "scales", (3, 1)), (readout, "scales", (1, 2)), (readout, "out", (1, 1)), (readout, "out", (2, 4)),
    (adjust, "repetition", (1,)), (adjust, "frequency", (3,)), (adjust, "presence", (1,)), (adjust, "bias", (9,)),
    (adjust, "bias", (1, 5)), (adjust, "bias", (1, 10)), (adjust, "out", (1, 1)), (adjust, "out", (2, 9)),
    (choose, "temperature", (1,)), (choose, "top_p", (3,)), (choose, "min_p", (1,)), (choose, "noise", (9,)),
    (choose, "noise", (1, 10)), (choose, "noise", (2, 9)),
])
def test_wrong_shapes_without_gradients_recorded(entries, call, name, shape, grad):
    """A size that does not fit is refused under no_grad too, whether or not the operand requires a gradient."""
    with torch.no_grad(), pytest.raises(ValueError, match=f"^{name} must have shape"):
        call(**{name: on_gpu(*shape, grad=grad)})
    assert entries.launched == 0


# The C boundary; addresses here are never read.
P = 1 << 30
READOUT = dict(x=P, x_dtype=7, x_stride=64, N=2, C=64, codes=2 * P, code_stride=32, scales=3 * P, scale_dtype=7,
               scale_stride=2, group=32, K=3, out=4 * P, out_dtype=7, out_stride=3, workspace=None, workspace_bytes=0,
               stream=None)


def entry(name, base, **wrong):
    return getattr(_lib.lib, name)(*{**base, **wrong}.values())


@pytest.mark.parametrize("wrong", [dict(x_stride=1 << 62), dict(x_stride=(1 << 61) + 64), dict(x_dtype=9, x_stride=1 << 62),
                                   dict(scale_stride=1 << 62), dict(scale_dtype=10, scale_stride=(1 << 62) + 2)])
def test_strides_whose_bytes_pass_64_bits(wrong):
    assert entry("ytm_readout", READOUT, **wrong) == _lib.YTM_EINVAL
    assert b"apart" in _lib.lib.ytm_last_error()


ADJUST = dict(scores=P, dtype=7, stride=8, N=2, V=8, tokens=2 * P, token_stride=4, T=4, lengths=None, prompt=None,
              repetition=None, frequency=None, presence=None, bias=3 * P, bias_stride=8, allowed=4 * P,
              allowed_stride=1, out=5 * P, out_dtype=7, out_stride=8, stream=None)


def test_history_whose_counts_pass_31_bits():
    assert entry("ytm_adjust_scores", ADJUST, T=1 << 31, token_stride=1 << 31, tokens=1 << 40) == _lib.YTM_EINVAL
    assert b"history" in _lib.lib.ytm_last_error()


@pytest.mark.parametrize("group", [2**64 + 32, 2**63, -32, 0, 33])
def test_groups_that_are_none(entries, group):
    with pytest.raises(ValueError, match="group"):
        readout(scales=on_gpu(3, 1), group=group)
    assert entries.launched == 0


CHOOSE = dict(scores=P, dtype=7, stride=8, N=2, V=8, temperature=2 * P, top_k=3 * P, top_p=4 * P, min_p=5 * P,
              noise=6 * P, noise_stride=8, tokens=7 * P, logprobs=8 * P, workspace=None, workspace_bytes=0, stream=None)
PENALTIES = dict(lengths=6 * P, prompt=7 * P, repetition=8 * P, frequency=9 * P, presence=10 * P)
SLICED = dict(V=100000, stride=100000, noise_stride=100000, workspace_bytes=1 << 30)
MANY = dict(N=20, x_stride=64, out_stride=3, workspace=9 * P, workspace_bytes=1 << 30)


@pytest.mark.parametrize("name,base,wrong", [
    ("ytm_readout", READOUT, dict(out=P)), ("ytm_readout", READOUT, dict(out=P + 4 * 127)),
    ("ytm_readout", READOUT, dict(out=P - 4 * 5)), ("ytm_readout", READOUT, dict(out=2 * P + 64)),
    ("ytm_readout", READOUT, dict(out=3 * P + 8)),
    ("ytm_readout", READOUT, dict(out=P + 4 * 64, x_stride=70, out_stride=70, N=3, K=7)),
    ("ytm_readout", READOUT, {**MANY, "workspace": P}), ("ytm_readout", READOUT, {**MANY, "workspace": 2 * P + 32}),
    ("ytm_readout", READOUT, {**MANY, "workspace": 3 * P - 16}), ("ytm_readout", READOUT, {**MANY, "out": 9 * P + 64}),
    # scores' own place, but of another size, distance, or one row for all; then a part of them
    ("ytm_adjust_scores", ADJUST, dict(out=P, out_dtype=9)), ("ytm_adjust_scores", ADJUST, dict(out=P, out_stride=9)),
    ("ytm_adjust_scores", ADJUST, dict(out=P, stride=0)), ("ytm_adjust_scores", ADJUST, dict(out=P + 4)),
    ("ytm_adjust_scores", ADJUST, dict(out=P + 4 * 15)), ("ytm_adjust_scores", ADJUST, dict(out=P - 4 * 15)),
    ("ytm_adjust_scores", ADJUST, dict(out=P + 4 * 8, stride=15, out_stride=15)),
    ("ytm_adjust_scores", ADJUST, dict(out=2 * P + 28)), ("ytm_adjust_scores", ADJUST, dict(out=3 * P + 60)),
    ("ytm_adjust_scores", ADJUST, dict(out=4 * P + 4)), ("ytm_adjust_scores", ADJUST, dict(out=3 * P, bias_stride=0)),
    *(("ytm_adjust_scores", dict(ADJUST, **PENALTIES), dict(out=p + 4)) for p in PENALTIES.values()),
    *(("ytm_choose", CHOOSE, {w: CHOOSE[r]}) for w in ("tokens", "logprobs")
      for r in ("scores", "temperature", "top_k", "top_p", "min_p", "noise")),
    ("ytm_choose", CHOOSE, dict(tokens=8 * P + 4)),
    *(("ytm_choose", dict(CHOOSE, **SLICED), dict(workspace=p)) for p in (P, 2 * P, 6 * P, 7 * P, 8 * P)),
])
def test_written_over_what_is_read(name, base, wrong):
    """Blocks run in no order, so one would read what another has written."""
    assert entry(name, base, **wrong) == _lib.YTM_EINVAL
    assert b"overlaps" in _lib.lib.ytm_last_error()


def dual(*shape):
    return forward_ad.make_dual(torch.zeros(*shape), torch.ones(*shape)).as_subclass(OnGpu)


@pytest.mark.parametrize("call,name,shape", FLOATS)
def test_operands_with_a_tangent(entries, call, name, shape):
    """Forward-mode derivatives would be dropped: refused, where they are recorded."""
    with forward_ad.dual_level():
        t = dual(*shape)
        with torch.no_grad(), pytest.raises(ValueError, match=f"^{name} .*tangent"):
            call(**{name: t})
        assert entries.launched == 0
        call()
        with torch.inference_mode():
            call(**{name: t})
        assert entries.launched == 2


@pytest.mark.parametrize("call,shape", [(readout, (2, 3)), (adjust, (2, 10))])
def test_outputs_count_as_changed(entries, call, shape):
    """A backward pass that has kept `out` sees that it was written to; one made in inference mode has no count."""
    out = on_gpu(*shape)
    for n in range(3):
        assert out._version == n
        assert call(out=out) is out
    with torch.inference_mode():
        call(out=on_gpu(*shape))
