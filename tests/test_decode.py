"""The answering operators (ytm_amd.decode): what runs on the host, and refusals that reach no
GPU."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from ytm_amd import _lib, decode  # noqa: E402

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def grid(w, scale):
    """The nearest value of the 4-bit grid, ties to the smaller magnitude, by trying all."""
    at = np.abs(np.abs(w / scale)[..., None] - VALUES)
    return np.sign(w) * VALUES[at.argmin(-1)] * scale


@pytest.mark.parametrize("C,K,group", [(1, 1, 32), (31, 3, 32), (32, 2, 64), (33, 5, 32), (200, 4, 64), (257, 3, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_packed_weights_are_the_nearest(C, K, group, dtype):
    w = np.random.default_rng(C).integers(-40, 41, (C, K)).astype(np.float32)
    w[: C // 3] = 0
    codes, scales = decode.pack_weights(w, group, dtype, device="cpu")
    assert codes.dtype == torch.uint8 and tuple(codes.shape) == (K, 16 * -(-C // 32)) and codes.is_contiguous()
    assert scales.dtype == dtype and tuple(scales.shape) == (K, -(-C // group))
    s = scales.double().numpy().repeat(group, 1)[:, :C].T
    got = decode.unpack_weights(codes, scales, C, group)
    assert got.shape == (C, K)
    # the values are products rounded to float32
    np.testing.assert_allclose(got, grid(w.astype(np.float64), s), rtol=1e-6, atol=0)


def test_packed_weights_exact_grid():
    """Weights that are a scale's multiples come back as they are."""
    v = np.concatenate([VALUES, -VALUES]) * 4
    w = np.random.default_rng(0).choice(v, (96, 7)).astype(np.float32)
    w[::32] = 24.0
    codes, scales = decode.pack_weights(w, 32, device="cpu")
    np.testing.assert_array_equal(decode.unpack_weights(codes, scales, 96), w)


@pytest.mark.parametrize("C", [1, 7, 8, 31, 32, 33, 100])
def test_packed_outputs(C):
    on = np.random.default_rng(C).integers(0, 2, (5, C)).astype(np.uint32)
    words = decode.pack_outputs(on, device="cpu")
    assert words.dtype == torch.int32 and tuple(words.shape) == (5, -(-C // 32))
    w = words.numpy().view(np.uint32)
    got = (w[:, np.arange(C) // 32] >> (np.arange(C) % 32).astype(np.uint32)) & 1
    np.testing.assert_array_equal(got, on)


@pytest.mark.parametrize("call", [
    lambda: decode.pack_weights(np.zeros(3, np.float32), device="cpu"),
    lambda: decode.pack_weights(np.zeros((3, 2), np.float32), group=16, device="cpu"),
    lambda: decode.pack_weights(np.zeros((3, 2), np.float32), group=48, device="cpu"),
    lambda: decode.pack_outputs(np.zeros(3, np.uint32), device="cpu"),
])
def test_host_refusals(call):
    with pytest.raises(ValueError):
        call()


def test_clause_banks_refused():
    class Banks:
        coalesced = False

    with pytest.raises(ValueError, match="banks"):
        decode.pack_model(Banks(), device="cpu")


def test_scale_type_refused():
    with pytest.raises(TypeError):
        decode.pack_weights(np.zeros((3, 2), np.float32), dtype=torch.float64, device="cpu")


def test_host_tensors_and_arrays_are_refused():
    x = torch.zeros(2, 4)
    for f in (decode.adjust_scores, decode.choose, lambda t: decode.readout(t, x, x)):
        with pytest.raises(ValueError, match="GPU"):
            f(x)
        with pytest.raises(TypeError, match="torch tensor"):
            f(x.numpy())


# The C boundary refuses before anything is launched; addresses here are never read.
P = 1 << 20
READOUT = dict(x=P, x_dtype=7, x_stride=64, N=2, C=64, codes=P, code_stride=32, scales=P, scale_dtype=7, scale_stride=2,
               group=32, K=3, out=P, out_dtype=7, out_stride=3, workspace=None, workspace_bytes=0, stream=None)
ADJUST = dict(scores=P, dtype=7, stride=8, N=2, V=8, tokens=P, token_stride=4, T=4, lengths=None, prompt=None,
              repetition=None, frequency=None, presence=None, bias=P, bias_stride=8, allowed=P, allowed_stride=1,
              out=P, out_dtype=7, out_stride=8, stream=None)
CHOOSE = dict(scores=P, dtype=7, stride=8, N=2, V=8, temperature=None, top_k=None, top_p=None, min_p=None, noise=P,
              noise_stride=8, tokens=P, logprobs=P, workspace=None, workspace_bytes=0, stream=None)


@pytest.mark.parametrize("function,base,wrong", [
    ("ytm_readout", READOUT, w) for w in (
        dict(x_dtype=8), dict(x_dtype=0), dict(scale_dtype=11), dict(out_dtype=11), dict(out_dtype=8), dict(N=-1),
        dict(N=65536), dict(C=-1), dict(K=-1), dict(C=1 << 31), dict(group=0), dict(group=16), dict(group=33),
        dict(x=None), dict(codes=None), dict(scales=None), dict(out=None), dict(codes=P + 8), dict(code_stride=40),
        dict(code_stride=16), dict(scale_stride=1), dict(x_stride=63), dict(out_stride=2),
        dict(C=2097121, x_stride=1 << 30, code_stride=1 << 30, scale_stride=1 << 30), dict(K=(1 << 23) + 1, out_stride=1 << 24), dict(code_stride=(8 << 20) + 16), dict(x_stride=(2 << 20) + 1),
        dict(scale_stride=(2 << 20) + 1),
        # a workspace that is missing, too small, at an odd address
        *(dict(C=200000, x_stride=200000, code_stride=100000, scale_stride=6250, **w) for w in (
            {}, dict(workspace=P, workspace_bytes=100), dict(workspace=P + 2, workspace_bytes=1 << 30))))
] + [
    ("ytm_adjust_scores", ADJUST, w) for w in (
        dict(dtype=11), dict(out_dtype=8), dict(N=-1), dict(N=65536), dict(V=-1), dict(V=(1 << 23) + 1), dict(T=-1),
        dict(scores=None), dict(out=None), dict(tokens=None), dict(stride=7), dict(out_stride=7), dict(token_stride=3),
        dict(bias_stride=7), dict(V=64, stride=64, out_stride=64, bias_stride=64, allowed_stride=1))
] + [
    ("ytm_choose", CHOOSE, w) for w in (
        dict(dtype=8), dict(N=-1), dict(V=-1), dict(V=(1 << 23) + 1), dict(scores=None), dict(tokens=None),
        dict(logprobs=None), dict(stride=7), dict(noise_stride=7),
        *(dict(V=100000, stride=100000, noise_stride=100000, **w) for w in (
            {}, dict(workspace=P, workspace_bytes=100), dict(workspace=P + 8, workspace_bytes=1 << 30))))
])
def test_boundary_refusals(function, base, wrong):
    assert getattr(_lib.lib, function)(*{**base, **wrong}.values()) == _lib.YTM_EINVAL
    assert _lib.lib.ytm_last_error()


@pytest.mark.parametrize("function,base", [("ytm_readout", dict(READOUT, N=0)), ("ytm_readout", dict(READOUT, K=0)),
                                           ("ytm_adjust_scores", dict(ADJUST, N=0)),
                                           ("ytm_adjust_scores", dict(ADJUST, V=0)), ("ytm_choose", dict(CHOOSE, N=0))])
def test_nothing_to_do(function, base):
    assert getattr(_lib.lib, function)(*base.values()) == _lib.YTM_OK


def test_workspace():
    n = ctypes.c_int64(-1)
    ask = _lib.lib.ytm_readout_workspace
    for wrong in ((8, 1, 1, 1, n), (7, -1, 1, 1, n), (7, 1, 2097121, 1, n), (7, 1, 1, -1, n), (7, 1, 1, 1, None)):
        assert ask(*wrong) == _lib.YTM_EINVAL
    for args in ((7, 0, 1000, 1), (7, 3, 0, 5), (7, 17, 7, 10), (11, 1, 10000, 10000), (7, 16, 256, 5)):
        assert ask(*args, n) == _lib.YTM_OK and n.value == 0
    for args in ((7, 16, 20000, 10), (11, 17, 8, 1)):
        assert ask(*args, n) == _lib.YTM_OK and n.value > 0


def test_choose_workspace():
    n = ctypes.c_int64(-1)
    ask = _lib.lib.ytm_choose_workspace
    for wrong in ((8, 1, 1, n), (7, -1, 1, n), (7, 1, -1, n), (7, 1, (1 << 23) + 1, n), (7, 1, 1, None)):
        assert ask(*wrong) == _lib.YTM_EINVAL
    for args in ((7, 0, 100000), (7, 3, 32767), (10, 1, 65535), (7, 65, 100000)):
        assert ask(*args, n) == _lib.YTM_OK and n.value == 0
    for args in ((7, 1, 32768), (9, 64, 65536)):
        assert ask(*args, n) == _lib.YTM_OK and n.value > 0
