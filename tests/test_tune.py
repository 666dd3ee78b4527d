"""What the adapting and learning operators refuse, before anything is launched.

Tensors here are on the CPU and say that they are on a GPU; the library's entries only count their
calls, so a call that is let through is seen and reads nothing.  The C entries get addresses that are never
read.
"""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as forward_ad  # noqa: E402

from ytm_amd import _lib, decode, tune  # noqa: E402


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
            self.launched += not name.endswith(("_workspace", "_table"))
            return 0

        return entry


@pytest.fixture
def entries(monkeypatch):
    e = Entries()
    monkeypatch.setattr(tune, "lib", e)
    monkeypatch.setattr(decode, "lib", e)
    monkeypatch.setattr(decode, "_device_now", lambda: 0)
    monkeypatch.setattr(decode, "_stream_of", lambda device: 0)
    return e


I32, F16, F64 = torch.int32, torch.float16, torch.float64
N, C, K, r, M, V, P = 4, 40, 6, 3, 2, 9, 2
ADAPT = dict(scores=on_gpu(N, K), x=on_gpu(N, 2, dtype=I32), down=on_gpu(M, r, C), up=on_gpu(M, K, r),
             which=on_gpu(N, dtype=I32), out=on_gpu(N, K))
GRADIENT = dict(grad=on_gpu(N, K), x=on_gpu(N, C), down=on_gpu(M, r, C), up=on_gpu(M, K, r),
                which=on_gpu(N, dtype=I32), hidden=on_gpu(N, r), out=(on_gpu(M, r, C), on_gpu(M, K, r)))
POLICY = dict(scores=on_gpu(N, V), tokens=on_gpu(N, dtype=I32), old=on_gpu(N), advantages=on_gpu(N), out=on_gpu(N, V))
PREFERENCE = dict(scores=on_gpu(N, V), tokens=on_gpu(N, dtype=I32), starts=on_gpu(2 * P + 1, dtype=I32),
                  reference=on_gpu(2 * P), out=on_gpu(N, V))
CALLS = {"adapt": (tune.adapt, ADAPT), "adapt_gradient": (tune.adapt_gradient, GRADIENT),
         "policy_loss": (tune.policy_loss, POLICY), "preference_loss": (tune.preference_loss, PREFERENCE)}


@pytest.mark.parametrize("name", list(CALLS))
def test_right_operands_pass(entries, name):
    function, base = CALLS[name]
    function(**base)
    assert entries.launched == 1


@pytest.mark.parametrize("name,operand,wrong,error", [
    ("adapt", "scores", np.zeros((N, K)), TypeError), ("adapt", "scores", on_gpu(N, K, dtype=F64), TypeError),
    ("adapt", "scores", on_gpu(N), ValueError), ("adapt", "scores", torch.zeros(N, K), ValueError),
    ("adapt", "scores", on_gpu(K, N).t(), ValueError), ("adapt", "scores", on_gpu(N, K, grad=True), ValueError),
    ("adapt", "x", on_gpu(N, 1, dtype=I32), ValueError), ("adapt", "x", on_gpu(N, C - 1), ValueError),
    ("adapt", "x", on_gpu(N - 1, C), ValueError), ("adapt", "x", on_gpu(N, C, dtype=F64), TypeError),
    ("adapt", "x", on_gpu(N, C, grad=True), ValueError), ("adapt", "x", on_gpu(C, N).t(), ValueError),
    ("adapt", "x", None, TypeError), ("adapt", "x", torch.zeros(N, C), ValueError),
    ("adapt", "down", on_gpu(M, r, C, dtype=F16), TypeError), ("adapt", "down", on_gpu(M, r + 1, C), ValueError),
    ("adapt", "down", on_gpu(r, C), ValueError), ("adapt", "down", on_gpu(M, C, r).transpose(1, 2), ValueError),
    ("adapt", "down", on_gpu(M, r, C, dtype=F64), TypeError), ("adapt", "down", on_gpu(M, r, C, grad=True), ValueError),
    ("adapt", "up", on_gpu(M, K, r, dtype=F16), TypeError), ("adapt", "up", on_gpu(M, r, K), ValueError),
    ("adapt", "up", on_gpu(M + 1, K, r), ValueError), ("adapt", "up", on_gpu(M, K, r, grad=True), ValueError),
    ("adapt", "up", None, TypeError), ("adapt", "which", None, TypeError),
    ("adapt", "which", on_gpu(N, dtype=torch.int64), TypeError), ("adapt", "which", on_gpu(N + 1, dtype=I32), ValueError),
    ("adapt", "hidden", on_gpu(N, r, dtype=F16), TypeError), ("adapt", "hidden", on_gpu(N, r + 1), ValueError),
    ("adapt", "hidden", on_gpu(r, N).t(), ValueError), ("adapt", "out", on_gpu(N, K + 1), ValueError),
    ("adapt", "out", on_gpu(N, K, dtype=F64), TypeError), ("adapt", "out", on_gpu(N, K, grad=True), ValueError),
    ("adapt_gradient", "grad", on_gpu(N, K, grad=True), ValueError), ("adapt_gradient", "grad", on_gpu(N, K + 1), ValueError),
    ("adapt_gradient", "hidden", None, TypeError), ("adapt_gradient", "hidden", on_gpu(N, r, dtype=F16), TypeError),
    ("adapt_gradient", "which", None, TypeError), ("adapt_gradient", "x", on_gpu(N, 1, dtype=I32), ValueError),
    ("adapt_gradient", "out", (on_gpu(M, r, C), on_gpu(M, K, r, dtype=F16)), TypeError),
    ("adapt_gradient", "out", (on_gpu(M, r, C + 1), on_gpu(M, K, r)), ValueError),
    ("adapt_gradient", "out", (on_gpu(M, C, r).transpose(1, 2), on_gpu(M, K, r)), ValueError),
    ("policy_loss", "scores", on_gpu(N, V, grad=True), ValueError), ("policy_loss", "tokens", None, TypeError),
    ("policy_loss", "tokens", on_gpu(N, dtype=torch.int64), TypeError), ("policy_loss", "old", on_gpu(N, dtype=F16), TypeError),
    ("policy_loss", "old", on_gpu(N + 1), ValueError), ("policy_loss", "old", on_gpu(N, grad=True), ValueError),
    ("policy_loss", "advantages", None, TypeError), ("policy_loss", "advantages", on_gpu(1), ValueError),
    ("policy_loss", "reference", on_gpu(N, 1), ValueError), ("policy_loss", "weights", on_gpu(N, dtype=F64), TypeError),
    ("policy_loss", "temperature", on_gpu(2), ValueError), ("policy_loss", "kl", 0.1, ValueError),
    ("policy_loss", "out", on_gpu(N + 1, V), ValueError), ("policy_loss", "out", on_gpu(N, V, dtype=F64), TypeError),
    ("preference_loss", "starts", on_gpu(2 * P, dtype=I32), ValueError), ("preference_loss", "starts", on_gpu(1, dtype=I32), ValueError),
    ("preference_loss", "starts", on_gpu(2 * P + 1), TypeError), ("preference_loss", "starts", None, TypeError),
    ("preference_loss", "reference", on_gpu(P), ValueError), ("preference_loss", "reference", None, TypeError),
    ("preference_loss", "tokens", None, TypeError), ("preference_loss", "temperature", on_gpu(N, dtype=F16), TypeError),
    ("preference_loss", "scores", on_gpu(V), ValueError), ("preference_loss", "out", torch.zeros(N, V), ValueError),
])
def test_wrong_operands_are_refused(entries, name, operand, wrong, error):
    function, base = CALLS[name]
    with pytest.raises(error):
        function(**{**base, operand: wrong})
    assert entries.launched == 0


@pytest.mark.parametrize("name,wrong", [("adapt", dict(scale=float("nan"))), ("adapt_gradient", dict(scale=float("inf"))),
                                        ("policy_loss", dict(kl=float("nan"))), ("policy_loss", dict(clip=float("inf"))),
                                        ("policy_loss", dict(clip_high=float("nan"))),
                                        ("preference_loss", dict(beta=float("inf"))),
                                        ("preference_loss", dict(smoothing=float("nan")))])
def test_numbers_that_are_not_finite_are_refused(entries, name, wrong):
    function, base = CALLS[name]
    with pytest.raises(ValueError, match="finite"):
        function(**{**base, **wrong})
    assert entries.launched == 0


@pytest.mark.parametrize("name,numbers", [("adapt", dict(scale=np.float32(2))), ("policy_loss", dict(clip=np.float32(0.1))),
                                          ("preference_loss", dict(beta=np.float64(0.1), smoothing=0))])
def test_numbers_of_other_kinds_pass(entries, name, numbers):
    function, base = CALLS[name]
    function(**{**base, **numbers})
    assert entries.launched == 1


@pytest.mark.parametrize("name", list(CALLS))
def test_tangents_are_refused(entries, name):
    function, base = CALLS[name]
    with forward_ad.dual_level():
        for operand, t in base.items():
            for i, one in enumerate(t if isinstance(t, tuple) else (t,)):
                if not one.is_floating_point() or (name, operand) == ("adapt_gradient", "down"):  # only its shape counts
                    continue
                dual = forward_ad.make_dual(one, torch.zeros_like(one))
                with pytest.raises(ValueError, match="tangent"):
                    function(**{**base, operand: dual if not isinstance(t, tuple) else t[:i] + (dual,) + t[i + 1:]})
    assert entries.launched == 0


@pytest.mark.parametrize("name", list(CALLS))
def test_what_is_written_counts_as_changed(entries, name):
    function, base = CALLS[name]
    out = base["out"] if isinstance(base["out"], tuple) else (base["out"],)
    if name == "adapt":
        hidden = on_gpu(N, r)
        base, out = dict(base, hidden=hidden), out + (hidden,)
    before = [t._version for t in out]
    function(**base)
    assert all(t._version > v for t, v in zip(out, before))


def test_adamw_refusals(entries):
    p, g = on_gpu(300), on_gpu(300)
    tune.AdamW([p], [g])
    for wrong, error in [
            (dict(parameters=[]), ValueError), (dict(gradients=[]), ValueError), (dict(bits=16), ValueError),
            (dict(parameters=[torch.zeros(300)]), ValueError), (dict(parameters=[np.zeros(300)]), TypeError),
            (dict(parameters=[on_gpu(300, dtype=F64)]), TypeError), (dict(gradients=[on_gpu(300, dtype=F16)]), TypeError),
            (dict(gradients=[on_gpu(299)]), ValueError), (dict(gradients=[on_gpu(300, grad=True)]), ValueError),
            (dict(parameters=[on_gpu(600)[::2]]), ValueError), (dict(gradients=[p]), ValueError),
            (dict(parameters=[on_gpu(1).expand(300)]), ValueError),
            (dict(states=dict(first=[on_gpu(300)])), ValueError),
            (dict(states=dict(first=[on_gpu(300)], second=[on_gpu(299)])), ValueError),
            (dict(states=dict(first=[], second=[on_gpu(300)])), ValueError),
            (dict(states=dict(first=[on_gpu(300)], second=[on_gpu(300, dtype=F16)])), TypeError),
            (dict(bits=8, states=dict(first=[on_gpu(300)], second=[on_gpu(300)])), ValueError),
            (dict(steps=torch.zeros(2, dtype=torch.int64)), ValueError), (dict(steps=torch.zeros(1)), ValueError)]:
        with pytest.raises(error):
            tune.AdamW(**{**dict(parameters=[p], gradients=[g]), **wrong})
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            tune.AdamW([forward_ad.make_dual(p, g)], [g])
    a = tune.AdamW([p], [g])
    launched = entries.launched
    for wrong in (dict(lr=float("nan")), dict(lr=on_gpu(2)), dict(lr=torch.tensor(0.1)), dict(eps=float("inf")),
                  dict(weight_decay=float("nan")), dict(active=on_gpu(2, dtype=torch.bool)), dict(lr=on_gpu(1, dtype=F16))):
        with pytest.raises(ValueError):
            a.step(**wrong)
    with pytest.raises(TypeError):
        a.step(active=on_gpu(1, dtype=I32))
    assert entries.launched == launched


def test_adamw_changes_versions(entries):
    p = on_gpu(300, grad=True)  # a leaf that autograd knows may be a parameter
    a = tune.AdamW([p], [on_gpu(300)])
    before = [t._version for t in (p, *a.first, *a.second)]
    a.step()
    assert all(t._version > v for t, v in zip((p, *a.first, *a.second), before))


@pytest.mark.parametrize("wrong", [dict(count=0), dict(clauses=0), dict(outputs=0), dict(rank=0), dict(rank=257),
                                   dict(scale=float("nan"))])
def test_adapters_refusals(wrong):
    with pytest.raises(ValueError):
        tune.Adapters(**{**dict(count=1, clauses=10, outputs=3, rank=2, device="cpu"), **wrong})
    with pytest.raises(TypeError):
        tune.Adapters(1, 10, 3, dtype=F64, device="cpu")


# The C boundary: addresses are never read.
A = 1 << 40


def at(i):
    return A + (i << 30)


C_ADAPT = dict(scores=at(0), dtype=7, stride=6, N=4, K=6, x=at(1), x_dtype=11, x_stride=2, C=40, down=at(2),
               down_adapter=120, down_rank=40, up=at(3), up_adapter=18, up_output=3, w_dtype=7, M=2, r=3, which=at(4),
               scale=1.0, hidden=at(5), hidden_stride=3, out=at(6), out_dtype=7, out_stride=6, workspace=at(7),
               workspace_bytes=1 << 20, stream=None)
C_GRADIENT = dict(grad=at(0), dtype=7, stride=6, N=4, K=6, x=at(1), x_dtype=11, x_stride=2, C=40, up=at(3), up_adapter=18,
                  up_output=3, w_dtype=7, M=2, r=3, which=at(4), scale=1.0, hidden=at(5), hidden_stride=3, d_down=at(6),
                  d_down_adapter=120, d_down_rank=40, d_up=at(7), d_up_adapter=18, d_up_output=3, workspace=at(8),
                  workspace_bytes=1 << 20, stream=None)
C_POLICY = dict(scores=at(0), dtype=7, stride=9, N=4, V=9, tokens=at(1), old=at(2), advantages=at(3), reference=at(4),
                kl=0.1, low=0.2, high=0.2, weights=at(5), temperature=at(6), losses=at(7), logprobs=at(8), grad=at(9),
                grad_dtype=7, grad_stride=9, workspace=None, workspace_bytes=0, stream=None)
C_PREFERENCE = dict(scores=at(0), dtype=7, stride=9, N=4, V=9, tokens=at(1), starts=at(2), pairs=2, reference=at(3),
                    beta=0.1, smoothing=0.1, temperature=at(4), losses=at(5), logprobs=at(6), grad=at(7), grad_dtype=7,
                    grad_stride=9, workspace=at(8), workspace_bytes=1 << 20, stream=None)
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("function,base,wrong", [
    ("ytm_adapt", C_ADAPT, w) for w in (
        dict(dtype=8), dict(dtype=11), dict(x_dtype=8), dict(w_dtype=11), dict(out_dtype=0), dict(N=-1), dict(N=65536),
        dict(K=-1), dict(K=(1 << 23) + 1), dict(C=-1), dict(C=2097121), dict(M=-1), dict(M=65536), dict(r=0), dict(r=257),
        dict(stride=5), dict(stride=-1), dict(x_stride=1), dict(down_rank=39), dict(down_adapter=39), dict(up_output=2),
        dict(up_adapter=2), dict(out_stride=5), dict(hidden_stride=2), dict(stride=1 << 62), dict(up_adapter=1 << 62),
        dict(out_stride=1 << 62), dict(scores=None), dict(x=None), dict(down=None), dict(up=None), dict(which=None),
        dict(out=None), dict(workspace=None), dict(workspace=at(7) + 4), dict(workspace_bytes=8), dict(scale=NAN),
        dict(scale=INF), dict(out=at(0) + 4), dict(out=at(1)), dict(out=at(2) + 400), dict(out=at(3)), dict(out=at(4)),
        dict(hidden=at(0)), dict(hidden=at(6)), dict(workspace=at(2)), dict(workspace=at(0), out=at(0)),
        dict(out=at(0), out_dtype=9), dict(out=at(0), out_stride=7), dict(hidden=at(1)))
] + [
    ("ytm_adapt_gradient", C_GRADIENT, w) for w in (
        dict(dtype=8), dict(x_dtype=8), dict(w_dtype=11), dict(N=-1), dict(N=65536), dict(K=-1), dict(C=-1), dict(M=65536),
        dict(r=0), dict(r=257), dict(stride=5), dict(x_stride=1), dict(d_down_rank=39), dict(d_down_rank=0),
        dict(d_down_adapter=119), dict(d_down_adapter=0), dict(d_up_output=2), dict(d_up_output=0), dict(d_up_adapter=17),
        dict(up_output=2), dict(hidden_stride=2), dict(grad=None), dict(x=None), dict(up=None), dict(which=None),
        dict(hidden=None), dict(d_down=None), dict(d_up=None), dict(workspace=None), dict(workspace=at(8) + 8),
        dict(workspace_bytes=8), dict(scale=NAN), dict(d_down=at(0)), dict(d_down=at(7)), dict(d_up=at(3)),
        dict(d_up=at(5)), dict(workspace=at(1)), dict(d_up_adapter=1 << 62), dict(d_up=at(4)))
] + [
    ("ytm_policy_loss", C_POLICY, w) for w in (
        dict(dtype=8), dict(grad_dtype=11), dict(N=-1), dict(N=65536), dict(V=-1), dict(V=(1 << 23) + 1), dict(stride=8),
        dict(grad_stride=8), dict(scores=None), dict(tokens=None), dict(old=None), dict(advantages=None),
        dict(reference=None), dict(losses=None), dict(logprobs=None), dict(grad=None), dict(kl=NAN), dict(kl=-0.1),
        dict(low=NAN), dict(low=-0.1), dict(low=1.1), dict(high=-0.1), dict(high=NAN), dict(grad=at(0) + 4),
        dict(grad=at(0), grad_dtype=9), dict(grad=at(0), grad_stride=10), dict(grad=at(1)), dict(grad=at(2)),
        dict(losses=at(0)), dict(losses=at(8)), dict(logprobs=at(2)), dict(logprobs=at(5)), dict(losses=at(9) + 16),
        *(dict(V=100000, stride=100000, grad_stride=100000, **w) for w in (
            {}, dict(workspace=at(10), workspace_bytes=8), dict(workspace=at(10) + 4, workspace_bytes=1 << 20),
            dict(workspace=at(0), workspace_bytes=1 << 20))))
] + [
    ("ytm_preference_loss", C_PREFERENCE, w) for w in (
        dict(dtype=8), dict(grad_dtype=11), dict(N=-1), dict(N=65536), dict(V=-1), dict(V=(1 << 23) + 1), dict(stride=8),
        dict(grad_stride=8), dict(scores=None), dict(tokens=None), dict(starts=None), dict(reference=None),
        dict(losses=None), dict(logprobs=None), dict(grad=None), dict(pairs=0), dict(pairs=65536), dict(beta=NAN),
        dict(beta=INF), dict(smoothing=-0.1), dict(smoothing=1.1), dict(smoothing=NAN), dict(workspace=None),
        dict(workspace_bytes=8), dict(workspace=at(8) + 4), dict(grad=at(0) + 4), dict(losses=at(2)), dict(logprobs=at(3)),
        dict(grad=at(2)), dict(losses=at(6)), dict(workspace=at(0)), dict(workspace=at(5)))
])
def test_boundary_refusals(function, base, wrong):
    assert getattr(_lib.lib, function)(*{**base, **wrong}.values()) == _lib.YTM_EINVAL
    assert _lib.lib.ytm_last_error()


@pytest.mark.parametrize("function,base", [("ytm_adapt", dict(C_ADAPT, N=0)), ("ytm_policy_loss", dict(C_POLICY, N=0)),
                                           ("ytm_adapt_gradient", dict(C_GRADIENT, M=0))])
def test_nothing_to_do(function, base):
    assert getattr(_lib.lib, function)(*base.values()) == _lib.YTM_OK


def test_workspaces():
    n = ctypes.c_int64(-1)
    for name, good, wrong in (
            ("adapt", (65535, 2097120, 65535, 256), ((-1, 1, 1, 1), (65536, 1, 1, 1), (1, -1, 1, 1), (1, 1, 65536, 1), (1, 1, 1, 0),
                                                     (1, 1, 1, 257))),
            ("adapt_gradient", (65535, 2097120, 1 << 23, 65535, 256), ((-1, 1, 1, 1, 1), (1, 1, 1 + (1 << 23), 1, 1), (1, 1, 1, -1, 1),
                                                                        (1, 1, 1, 1, 0), (1, 2097121, 1, 1, 1))),
            ("policy_loss", (1, 1 << 23), ((-1, 1), (65536, 1), (1, -1), (1, 1 + (1 << 23)))),
            ("preference_loss", (65535, 1 << 23), ((-1, 1), (65536, 1), (1, -1), (1, 1 + (1 << 23))))):
        ask = getattr(_lib.lib, f"ytm_{name}_workspace")
        assert ask(*good, n) == _lib.YTM_OK and n.value > 0
        assert ask(*good, None) == _lib.YTM_EINVAL
        for args in wrong:
            assert ask(*args, n) == _lib.YTM_EINVAL


def tensors(*counts, **kw):
    rows = (_lib.AdamWTensor * len(counts))()
    for row, n in zip(rows, counts):
        for name, v in {**dict(parameter=A, gradient=A, first=A, second=A, first_scales=A, second_scales=A, count=n,
                               parameter_dtype=7, gradient_dtype=7), **kw}.items():
            setattr(row, name, v)
    return rows


def test_adamw_table():
    size, chunks = ctypes.c_int64(), ctypes.c_int64()
    make = _lib.lib.ytm_adamw_table
    assert make(tensors(1, 4096, 0, 5000), 4, 8, None, size, chunks) == _lib.YTM_OK
    assert size.value > 0 and chunks.value >= 3
    host = (ctypes.c_ubyte * (size.value + 8))(*([77] * (size.value + 8)))
    assert make(tensors(1, 4096, 0, 5000), 4, 8, host, size, chunks) == _lib.YTM_OK
    assert bytes(host[size.value:]) == bytes([77] * 8)
    assert make(None, 0, 32, None, size, chunks) == _lib.YTM_OK and chunks.value == 0
    for rows, bits in ((tensors(5), 16), (tensors(-1), 32), (tensors(5, parameter_dtype=8), 32),
                       (tensors(5, gradient_dtype=9), 32), (tensors(5, parameter=None), 32), (tensors(5, gradient=None), 32),
                       (tensors(5, second=None), 32), (tensors(5, first_scales=None), 8), (tensors(1 << 50), 32)):
        assert make(rows, len(rows), bits, None, size, chunks) == _lib.YTM_EINVAL
    assert make(tensors(5), 1, 32, None, None, chunks) == _lib.YTM_EINVAL
    assert make(tensors(5, first_scales=None, second_scales=None), 1, 32, None, size, chunks) == _lib.YTM_OK


@pytest.mark.parametrize("wrong", [dict(n=-1), dict(chunks=-1), dict(bits=16), dict(table=None), dict(table=A + 8),
                                   dict(steps=None), dict(beta1=1.0), dict(beta1=NAN), dict(beta2=-0.1), dict(eps=-1.0),
                                   dict(eps=NAN), dict(chunks=1 << 40)])
def test_adamw_boundary_refusals(wrong):
    base = dict(table=A, n=1, chunks=1, bits=32, steps=A, active=None, rate=0.1, rate_at=None, beta1=0.9, beta2=0.99,
                eps=1e-8, decay=0.0, seed=0, stream=None)
    assert _lib.lib.ytm_adamw(*{**base, **wrong}.values()) == _lib.YTM_EINVAL
