"""Weights that their scales' type cannot hold as the largest weight over six."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from ytm_amd import decode  # noqa: E402

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# least positive number of the type
LEAST = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}


def groups(*largest, outputs=2):
    """(32 clauses a group, outputs): each group's weights from its largest down, both signs."""
    w = np.linspace(1, -1, 32)[:, None] * np.ones(outputs)
    return np.concatenate([np.float64(v) * w for v in largest]).astype(np.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_codes_are_nearest_at_every_size(dtype):
    """Down to the least positive scale, from which on weights take smaller codes; groups of zeros stay."""
    for e in range(-149, 126, 3):
        w = groups(2.0**e, 0.0, 1.0)
        if 2.0**e / 6 > torch.finfo(dtype).max:
            continue
        codes, scales = decode.pack_weights(w, 32, dtype, device="cpu")
        s = scales.double().numpy()
        assert (s > 0).all() and np.isfinite(s).all() and (s[:, 1] == 1).all()
        code = np.stack((codes.numpy() & 15, codes.numpy() >> 4), 2).reshape(2, 96)
        got = np.where(code & 8, -1, 1) * VALUES[code & 7] * s.repeat(32, 1)
        # by trying all: no value of the grid is nearer
        off = np.abs(np.abs(w.T.astype(np.float64))[..., None] - VALUES * s.repeat(32, 1)[..., None]).min(-1)
        np.testing.assert_array_equal(np.abs(got - w.T), off, err_msg=str(e))
        assert (np.sign(got) * np.sign(w.T) >= 0).all()
        assert (np.abs(s[:, 0] - 2.0**e / 6) <= np.maximum(2.0**e / 6 * 2.0**-8, LEAST[dtype])).all()


@pytest.mark.parametrize("dtype,weight", [(torch.float16, 6 * 65520.0), (torch.float16, 500000.0),
                                          (torch.float16, 3e38), (torch.float32, np.inf), (torch.float32, -np.inf),
                                          (torch.float16, np.nan), (torch.bfloat16, np.nan)])
def test_weights_past_the_scales_type(dtype, weight):
    w = np.ones((40, 3), np.float32)
    w[35, 1] = weight
    with pytest.raises(ValueError, match="float16|finite"):
        decode.pack_weights(w, 32, dtype, device="cpu")


@pytest.mark.parametrize("dtype", TYPES)
def test_the_largest_weights(dtype):
    top = 6 * 65504.0 if dtype == torch.float16 else 3e38  # six times whose rounded scale float32 holds
    codes, scales = decode.pack_weights(groups(top), 32, dtype, device="cpu")
    assert bool(torch.isfinite(scales).all())
    np.testing.assert_allclose(decode.unpack_weights(codes, scales, 32)[0], top, rtol=2.0**-8)


def test_weights_past_float32():
    with pytest.raises(ValueError, match="finite"):
        decode.pack_weights(np.full((32, 1), 1e39), device="cpu")
