"""What AdamW and Adapters make of their surroundings and of what they are given, without a GPU: tensors that say that
they are on one, and entries that count their calls (as in test_tune.py)."""
import copy
import io
import pickle

import pytest

torch = pytest.importorskip("torch")

from ytm_amd import _lib, tune  # noqa: E402

from test_tune import C_GRADIENT, F16, GRADIENT, I32, OnGpu, entries, on_gpu  # noqa: E402, F401


def test_tables_are_made_on_the_host(entries):  # noqa: F811
    p, g = on_gpu(300), on_gpu(300)
    with torch.device("meta"):
        a = tune.AdamW([p], [g])
    assert a._table.device.type == "cpu"


@pytest.mark.parametrize("which", [None, 3, torch.zeros((), dtype=I32), on_gpu(4, 1, dtype=I32)])
def test_adapters_say_what_is_wrong(entries, which):  # noqa: F811
    a = object.__new__(tune.Adapters)
    a.scale, a.down, a.up = 1.0, on_gpu(2, 3, 40), on_gpu(2, 6, 3)
    with pytest.raises((TypeError, ValueError), match="which"):
        a.adapt(on_gpu(4, 6), on_gpu(4, 2, dtype=I32), which)
    assert entries.launched == 0


class Copied(OnGpu):
    def __deepcopy__(self, memo):
        return memo.setdefault(id(self), self.clone())


def copied_on_gpu(n, dtype=torch.float32):
    return on_gpu(n, dtype=dtype).as_subclass(Copied)


def addresses(a):
    """The parameters' addresses in an AdamW's table, whose rows are 136 bytes or more, each parameter's first."""
    words = a._table[:a._table.numel() // 8 * 8].view(torch.int64).tolist()
    return [t.data_ptr() in words for t in (*a.parameters, *a.gradients, *a.first, *a.second)], words


def saved(a):
    f = io.BytesIO()
    torch.save(a, f)
    f.seek(0)
    return torch.load(f, weights_only=False)  # what this test wrote itself


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("copied", [copy.deepcopy, lambda a: pickle.loads(pickle.dumps(a)), saved])
def test_copies_have_addresses_of_their_own(copied, bits):
    sizes, state = (300, 7), torch.float32 if bits == 32 else torch.float8_e4m3fn
    states = {name: [copied_on_gpu(n, dtype=state) for n in sizes] for name in ("first", "second")}
    if bits == 8:
        states |= {name: [copied_on_gpu(-(-n // 256)) for n in sizes] for name in ("first_scales", "second_scales")}
    a = tune.AdamW([copied_on_gpu(n) for n in sizes], [copied_on_gpu(n) for n in sizes], bits=bits, states=states, steps=5, seed=3)
    b = copied(a)
    assert (b.bits, b.seed, b.steps.tolist()) == (bits, 3, [5, 5])
    for one, other in ((a, b), (b, a)):
        there, words = addresses(one)
        assert all(there)
        assert not any(t.data_ptr() in words for t in (*other.parameters, *other.gradients, *other.first, *other.second))
    b.steps.add_(1)
    assert a.steps.tolist() == [5, 5]
    c = copy.copy(a)
    assert all(addresses(c)[0]) and c.parameters[0] is a.parameters[0] and c.steps is a.steps


@pytest.mark.parametrize("steps", [-1, torch.tensor([0, -1]), torch.tensor([-(2**40), 3])])
def test_steps_before_the_first_are_refused(entries, steps):  # noqa: F811
    with pytest.raises(ValueError, match="0 or more"):
        tune.AdamW([on_gpu(3), on_gpu(4)], [on_gpu(3), on_gpu(4)], steps=steps)
    tune.AdamW([on_gpu(3), on_gpu(4)], [on_gpu(3), on_gpu(4)], steps=torch.tensor([0, 2**40]))


BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("w,kinds,error", [(F16, (F16, F16), None), (F16, (F32, F32), None), (BF16, (F32, F32), None),
                                           (F32, (F32, F32), None), (F16, (F32, F16), TypeError),
                                           (F16, (F16, F32), TypeError), (F16, (BF16, BF16), TypeError),
                                           (F32, (F16, F16), TypeError)])
def test_types_of_adapters_gradients(entries, w, kinds, error):  # noqa: F811
    down, up = (on_gpu(*GRADIENT[t].shape, dtype=w) for t in ("down", "up"))
    operands = {**GRADIENT, "down": down, "up": up, "out": (on_gpu(*down.shape, dtype=kinds[0]), on_gpu(*up.shape, dtype=kinds[1]))}
    if error:
        with pytest.raises(error):
            tune.adapt_gradient(**operands)
        assert entries.launched == 0
    else:
        assert tune.adapt_gradient(**operands)[0].dtype is kinds[0] and entries.launched == 1


@pytest.mark.parametrize("w,d", [(7, 9), (9, 10), (10, 9), (9, 11), (7, 8)])
def test_types_of_adapters_gradients_at_the_boundary(w, d):
    operands = {}
    for name, v in dict(C_GRADIENT, w_dtype=w).items():
        if name == "d_down":
            operands["d_dtype"] = d
        operands[name] = v
    assert _lib.lib.ytm_adapt_gradient_as(*operands.values()) == _lib.YTM_EINVAL
    # where the wider gradients reach what a narrower one would not
    operands |= dict(w_dtype=9, d_dtype=7, d_down=C_GRADIENT["d_up"] - 4 * 200)
    assert _lib.lib.ytm_adapt_gradient_as(*operands.values()) == _lib.YTM_EINVAL
    assert b"overlap" in _lib.lib.ytm_last_error()


def adapters(monkeypatch, count):
    """Adapters whose optimiser only notes which of its tensors it should step, and these notes."""
    a, said = object.__new__(tune.Adapters), []
    a.count, a.scale, a.down, a.up = count, 1.0, on_gpu(count, 2, 3), on_gpu(count, 5, 2)
    a.gradients = on_gpu(count, 2, 3), on_gpu(count, 5, 2)
    parameters, gradients = a._each()
    a.optimizer = type("Optimizer", (), {"step": lambda self, *args, active: said.append(active)})()
    a.optimizer.parameters, a.optimizer.gradients = parameters, gradients
    monkeypatch.setattr(tune, "adapt_gradient", lambda *args, **kw: None)
    return a, said


@pytest.mark.parametrize("which", [[], [0], [3, 0, 3, 3], [-1, 4, 2**31 - 1, -(2**31), 1], [-5, 9]])
def test_adapters_step_those_that_a_batch_names(monkeypatch, which):
    a, said = adapters(monkeypatch, 4)
    a.learn(None, None, torch.tensor(which, dtype=I32), None)
    assert said[0].dtype is torch.bool and said[0].is_contiguous()
    assert said[0].tolist() == [n in which for n in range(4) for _ in range(2)]


def test_adapters_find_those_named_without_a_table_of_rows_and_adapters(monkeypatch):
    """As many rows and adapters as the entries take: what it needs is counted in either, not in their product."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Sizes(TorchDispatchMode):
        largest = 0

        def __torch_dispatch__(self, function, types, args=(), kwargs=None):
            out = function(*args, **(kwargs or {}))
            for t in out if isinstance(out, (tuple, list)) else (out,):
                if isinstance(t, torch.Tensor):
                    Sizes.largest = max(Sizes.largest, t.numel())
            return out

    a, _ = adapters(monkeypatch, 3000)
    which = torch.arange(5000, dtype=I32)
    with Sizes():
        a.learn(None, None, which, None)
    assert Sizes.largest <= 2 * (3000 + 2) + 5000


def test_a_step_takes_the_tensors_of_its_table(monkeypatch):
    """Also where somebody has put more into the lists, of which it has no rows."""
    calls = []
    monkeypatch.setattr(tune, "_call", lambda function, device, *args: calls.append(args))
    a = tune.AdamW([on_gpu(3), on_gpu(4)], [on_gpu(3), on_gpu(4)])
    a.parameters.append(on_gpu(5))
    a.step()
    assert calls[0][1] == 2
    with pytest.raises(ValueError, match="active"):
        a.step(active=on_gpu(3, dtype=torch.bool))


@pytest.mark.parametrize("steps,error", [(torch.zeros(2, dtype=torch.int64), ValueError), (on_gpu(2, dtype=I32), TypeError),
                                         (on_gpu(3, dtype=torch.int64), ValueError), (3, TypeError), (None, TypeError),
                                         (on_gpu(4, dtype=torch.int64)[::2], ValueError)])
def test_steps_that_a_step_cannot_count_are_refused(entries, steps, error):  # noqa: F811
    a = tune.AdamW([on_gpu(3), on_gpu(4)], [on_gpu(3), on_gpu(4)])
    was = a.steps
    with pytest.raises(error, match="steps"):
        a.steps = steps
    assert a.steps is was
    a.steps = good = on_gpu(2, dtype=torch.int64)
    assert a.steps is good


@pytest.mark.parametrize("name", ["down", "up", "gradients"])
def test_adapters_refuse_tensors_that_their_optimiser_does_not_step(monkeypatch, name):
    a, said = adapters(monkeypatch, 3)
    which = torch.zeros(2, dtype=I32)
    a.learn(None, None, which, None)
    held = getattr(a, name)
    setattr(a, name, tuple(t.clone() for t in held) if isinstance(held, tuple) else held.clone())
    with pytest.raises(ValueError, match="copy into"):
        a.learn(None, None, which, None)
    assert len(said) == 1
    a.optimizer.parameters, a.optimizer.gradients = a._each()  # one that does
    a.learn(None, None, which, None)
    assert len(said) == 2
