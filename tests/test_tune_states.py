"""What AdamW and Adapters make of their surroundings and of what they are given, without a GPU: tensors that say that
they are on one, and entries that count their calls (as in test_tune.py)."""
import pytest

torch = pytest.importorskip("torch")

from ytm_amd import tune  # noqa: E402

from test_tune import I32, entries, on_gpu  # noqa: E402, F401


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
