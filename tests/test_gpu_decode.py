"""The answering operators on the GPU against plain numpy in 64 bits.

Where every product and sum is a whole number of a power of two that float32 holds, results have
to be equal.  Elsewhere the bounds are those of the roundings made: a float32 sum of products
that are exact, in parts of at most `depth` terms one after the other, is within
depth 2^-23 sum |terms| (twice the bound of rounding to nearest, for an adder that cuts), and an
output of 8 or 11 bits of fraction within half of its last one.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ytm_amd = pytest.importorskip("ytm_amd")
from ytm_amd import decode  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a unit in the last place, relative, and the least difference of numbers near zero
ROUND = {"f32": (2.0**-24, 2.0**-149), "f16": (2.0**-11, 2.0**-25), "bf16": (2.0**-8, 2.0**-133)}
VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6])


def host(t):
    return t.detach().double().cpu().numpy()


def spread(t, pad, offset=0):
    """The same tensor (rows, width) with its rows `pad` elements further apart, off by `offset`."""
    if pad == 0 and offset == 0:
        return t
    rows, width = t.shape
    big = torch.full((rows * (width + pad) + offset,), 77, dtype=t.dtype, device=t.device)
    out = big[offset:].view(rows, width + pad)[:, :width]
    out.copy_(t)
    return out


# -------------------------------------------------------------------------------- readout
def weights(rng, C, K, group, scale, exact):
    codes = rng.integers(0, 256, (K, 16 * -(-C // 32)), dtype=np.uint8)
    groups = -(-C // group)
    s = 2.0 ** rng.integers(-2, 3, (K, groups)) if exact else rng.uniform(0.01, 3.0, (K, groups))
    scales = torch.from_numpy(s.astype(np.float32)).to(TYPES[scale])
    code = np.stack((codes & 15, codes >> 4), 2).reshape(K, -1)[:, :C]
    return codes, scales, VALUES[code] * host(scales).repeat(group, 1)[:, :C]


def clause_rows(rng, N, C, x, exact):
    """(tensor, its values)"""
    if x == "bits":
        on = (rng.random((N, C)) < 0.3).astype(np.uint32)
        words = decode.pack_outputs(on)
        if C % 32:  # bits past the last clause are ignored
            words[:, -1] |= -(1 << C % 32)
        return words, on.astype(np.float64)
    v = rng.integers(-4, 5, (N, C)).astype(np.float32) if exact else rng.normal(0, 2, (N, C)).astype(np.float32)
    t = torch.from_numpy(v).to(TYPES[x]).cuda()
    return t, host(t)


SIZES = [(1, 1, 1), (1, 31, 5), (1, 32, 16), (2, 33, 17), (3, 128, 1), (15, 64, 15), (16, 127, 16), (17, 129, 33),
         (33, 300, 40), (64, 512, 64), (70, 1000, 50), (129, 257, 130), (200, 96, 300), (1, 20000, 10), (1, 700, 1000),
         (5, 4097, 300), (1, 2000, 5000)]


@pytest.mark.parametrize("x", ["bits", "f32", "f16", "bf16"])
@pytest.mark.parametrize("N,C,K", SIZES)
def test_readout_exact(N, C, K, x):
    """Small whole numbers and scales of powers of two: every sum is exact."""
    rng = np.random.default_rng(N + 7 * C + 13 * K)
    for group in (32, 64, 96, 128, 256):
        codes, scales, w = weights(rng, C, K, group, "f32", True)
        xt, xv = clause_rows(rng, N, C, x, True)
        got = decode.readout(xt, torch.from_numpy(codes).cuda(), scales.cuda(), group=group, clauses=C)
        np.testing.assert_array_equal(host(got), xv @ w.T, err_msg=f"group {group}")


def depth(C, group):
    return 64 + C // 32


@pytest.mark.parametrize("x,scale,out", [("bits", "f32", "f32"), ("bits", "f16", "bf16"), ("f32", "f32", "f32"),
                                         ("f32", "bf16", "f16"), ("f16", "f16", "f32"), ("f16", "f32", "f16"),
                                         ("bf16", "bf16", "f32"), ("bf16", "f16", "bf16")])
@pytest.mark.parametrize("N,C,K,group", [(1, 500, 40, 32), (7, 1000, 33, 64), (40, 777, 129, 128), (150, 1024, 100, 32),
                                         (300, 333, 65, 64), (2, 9000, 20, 512)])
def test_readout_types(N, C, K, group, x, scale, out):
    rng = np.random.default_rng(N + C)
    codes, scales, w = weights(rng, C, K, group, scale, False)
    xt, xv = clause_rows(rng, N, C, x, False)
    to = torch.empty(N, K, dtype=TYPES[out], device="cuda")
    got = decode.readout(xt, torch.from_numpy(codes).cuda(), scales.cuda(), group=group, clauses=C, out=to)
    assert got is to
    want, size = xv @ w.T, np.abs(xv) @ np.abs(w).T
    rel, least = ROUND[out]
    err = np.abs(host(got) - want)
    assert (err <= depth(C, group) * 2.0**-23 * size + rel * np.abs(want) + least).all(), err.max()


@pytest.mark.parametrize("x,pad,offset", [("f32", 3, 1), ("f16", 5, 1), ("bf16", 1, 3), ("bits", 2, 1), ("f16", 8, 8)])
@pytest.mark.parametrize("N", [4, 90])
def test_readout_strides(x, pad, offset, N):
    rng = np.random.default_rng(N)
    C, K = 333, 70
    codes, scales, w = weights(rng, C, K, 32, "f16", True)
    xt, xv = clause_rows(rng, N, C, x, True)
    wide = torch.zeros(K, codes.shape[1] + 32, dtype=torch.uint8, device="cuda")
    wide[:, 16:-16] = torch.from_numpy(codes).cuda()
    to = spread(torch.zeros(N, K, device="cuda"), 5, 3)
    whole = to.as_strided((N * (K + 5),), (1,), 3)
    decode.readout(spread(xt, pad, offset), wide[:, 16:-16], spread(scales.cuda(), 3, 1), group=32, clauses=C, out=to)
    np.testing.assert_array_equal(host(to), xv @ w.T)
    left = whole.view(N, K + 5)[:, K:]
    assert bool((left == 77).all()), "written past a row's end"


def test_readout_infinities_stay_in_their_row():
    rng = np.random.default_rng(3)
    N, C, K = 20, 200, 48
    codes, scales, w = weights(rng, C, K, 32, "f32", True)
    codes = codes & 0x77 | 0x11  # positive, no zeros
    w = VALUES[np.stack((codes & 15, codes >> 4), 2).reshape(K, -1)[:, :C]] * host(scales).repeat(32, 1)[:, :C]
    for x in ("f32", "f16", "bf16"):
        xt, xv = clause_rows(rng, N, C, x, True)
        for row, v in ((3, np.inf), (9, -np.inf), (17, np.nan)):
            xt[row, 77] = v
            xv[row, 77] = v
        got = host(decode.readout(xt, torch.from_numpy(codes).cuda(), scales.cuda()))
        np.testing.assert_array_equal(got, xv @ w.T, err_msg=x)


def test_readout_large_and_small_values():
    """float32 values over its whole range keep their 24 bits."""
    rng = np.random.default_rng(4)
    N, C, K = 6, 64, 32
    codes, scales, w = weights(rng, C, K, 32, "f32", True)
    for e in (-100, -40, 0, 40, 100):
        v = (rng.integers(1, 1 << 24, (N, 1)) * 2.0**e * 2.0**-24).astype(np.float32)
        xv = np.zeros((N, C), np.float32)
        at = rng.integers(0, C, N)
        xv[np.arange(N), at] = v[:, 0]
        got = host(decode.readout(torch.from_numpy(xv).cuda(), torch.from_numpy(codes).cuda(), scales.cuda()))
        want = xv.astype(np.float64) @ w.T
        # one term of up to 3 more bits of fraction, in up to three parts
        assert (np.abs(got - want) <= 4 * 2.0**-24 * np.abs(want)).all()


def test_readout_no_clauses():
    to = torch.full((3, 5), 9.0, device="cuda")
    decode.readout(torch.empty(3, 0, device="cuda"), torch.empty(5, 0, dtype=torch.uint8, device="cuda"),
                   torch.empty(5, 0, device="cuda"), out=to)
    assert bool((to == 0).all())


def test_readout_of_a_model():
    """Class sums through packed weights are those of the weights the codes stand for."""
    from ytm_amd import MultiClassTM

    C, K = 300, 10
    tm = MultiClassTM(C, 50, 5.0, (60, 1, 1), K, seed=3)
    rng = np.random.default_rng(8)
    ta = np.where(rng.random((C, tm.number_of_literals)) < 2 / tm.number_of_literals, 200, 60).astype(np.uint32)
    w = (rng.choice(VALUES, (C, K)) * 8).astype(np.float32)
    w[::32] = 48.0
    tm.load_state_dict({"state": {"ta_state": ta, "clause_weights": w, "min_y": None, "max_y": None,
                                  "patch_weights": np.zeros((C, 1), np.int32)}})
    X = rng.integers(0, 2, (40, 60)).astype(np.uint32)
    codes, scales = decode.pack_model(tm)
    got = decode.readout(decode.pack_outputs(tm.transform(X)), codes, scales, clauses=C)
    np.testing.assert_array_equal(got.cpu().numpy(), tm.score(tm.encode(X), True))


def test_example_goes_on_writing():
    """The example's steps together: the grammar holds, and training shows."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import next_word

    tm, after = next_word.train(samples=6000, epochs=3)
    said = next_word.write(tm, texts=5, length=12)
    assert said.shape == (5, 12 + next_word.CONTEXT) and (said >= 0).all() and (said < next_word.WORDS).all()
    stops = said == next_word.STOP
    assert not (stops[:, 1:] & stops[:, :-1]).any()
    follows = (after[said[:, next_word.CONTEXT - 1:-1]] == said[:, next_word.CONTEXT:, None]).any(2)
    assert follows.mean() > 0.5  # 4 of 60 words do
    np.testing.assert_array_equal(said, next_word.write(tm, texts=5, length=12))


# --------------------------------------------------------------------------- adjust_scores
def shaped(x, tokens, lengths, prompt, rep, freq, pres, bias, allowed):
    """(result, magnitude of its terms) in 64 bits, by the definition."""
    N, V = x.shape
    s, size = x.astype(np.float64).copy(), np.abs(np.where(np.isfinite(x), x, 0)).astype(np.float64)
    for n in range(N):
        told = set()
        count = {}
        for i, t in enumerate(tokens[n][:max(0, lengths[n])] if tokens is not None else []):
            if 0 <= t < V:
                told.add(int(t))
                if i >= prompt[n]:
                    count[int(t)] = count.get(int(t), 0) + 1
        for t in told:
            s[n, t] = s[n, t] / rep[n] if s[n, t] > 0 else s[n, t] * rep[n]
            size[n, t] *= max(rep[n], 1 / rep[n])
            if t in count:
                s[n, t] -= freq[n] * count[t] + pres[n]
                size[n, t] += freq[n] * count[t] + abs(pres[n])
    if bias is not None:
        s += bias
        size += np.abs(bias)
    if allowed is not None:
        s[np.broadcast_to(~allowed, s.shape)] = -np.inf
    return s, size


def words_of(bits):
    return decode.pack_outputs(bits)


def adjust_case(N, V, T, seed, x="f32", out="f32", bias="rows", allowed="rows", kind="zipf", pad=0, offset=0):
    rng = np.random.default_rng(seed)
    xt = torch.from_numpy(rng.normal(0, 4, (N, V)).astype(np.float32)).to(TYPES[x]).cuda()
    if kind == "zipf":
        tokens = np.minimum(V ** rng.random((N, T)), V - 1).astype(np.int32)
    elif kind == "one":
        tokens = np.full((N, T), rng.integers(0, V), np.int32)
    else:  # strays: padding, numbers past the vocabulary
        tokens = rng.choice(np.array([-1, -2**31, V, V + 5, 2**31 - 1, 0, V - 1], np.int64), (N, T)).astype(np.int32)
    lengths = rng.integers(-1, T + 3, N).astype(np.int32)
    lengths[0] = T
    prompt = (rng.random(N) * (T + 2)).astype(np.int32) - 1
    rep, freq, pres = (rng.uniform(a, b, N).astype(np.float32) for a, b in ((0.5, 2), (0, 1), (-1, 1)))
    b = None if bias == "none" else rng.normal(0, 2, (V,) if bias == "shared" else (N, V)).astype(np.float32)
    ok = None if allowed == "none" else rng.random((1 if allowed == "shared" else N, V)) < 0.5
    if ok is not None and allowed == "rows" and N > 1:
        ok[N // 2] = False  # a row the grammar leaves nothing
    to = spread(torch.zeros(N, V, dtype=TYPES[out], device="cuda"), pad, offset)
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    words = None if ok is None else words_of(ok)
    got = decode.adjust_scores(
        spread(xt, pad, offset), tokens=spread(dev(tokens), pad, offset) if T else dev(tokens), lengths=dev(lengths),
        prompt=dev(prompt), repetition=dev(rep), frequency=dev(freq), presence=dev(pres),
        bias=None if b is None else (spread(dev(b), pad, offset) if b.ndim == 2 else dev(b)),
        allowed=words if words is None or allowed == "rows" else words[0].contiguous(), out=to)
    assert got is to
    want, size = shaped(host(xt), tokens, lengths, prompt, rep.astype(np.float64), freq.astype(np.float64),
                        pres.astype(np.float64), None if b is None else b.astype(np.float64), ok)
    g = host(got)
    np.testing.assert_array_equal(np.isneginf(g), np.isneginf(want))
    fine = np.isfinite(want)
    rel, least = ROUND[out]
    # up to five roundings to float32, then the output's
    bound = 5 * 2.0**-24 * size + rel * np.abs(np.where(fine, want, 0)) + least
    assert (np.abs(g[fine] - want[fine]) <= bound[fine]).all()


@pytest.mark.parametrize("V", [1, 31, 32, 33, 100, 1023, 4095, 4096, 4097, 8200, 20001])
@pytest.mark.parametrize("N,T,kind", [(1, 0, "zipf"), (1, 1, "zipf"), (3, 150, "zipf"), (2, 4096, "one"), (3, 700, "stray")])
def test_adjust_sizes(N, V, T, kind):
    adjust_case(N, V, T, N + V + T, kind=kind)


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bias,allowed", [("none", "none"), ("shared", "shared"), ("rows", "none"), ("none", "rows")])
def test_adjust_types(x, out, bias, allowed):
    adjust_case(5, 5000, 300, 1, x, out, bias, allowed)


@pytest.mark.parametrize("x,out", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (8, 2), (5, 7)])
def test_adjust_strides(x, out, pad, offset):
    adjust_case(4, 4501, 90, pad, x, out, pad=pad, offset=offset)


def test_adjust_in_place_and_untouched():
    """Without a history, bias or grammar scores come back as they are, NaN and infinities too."""
    x = torch.randn(3, 999, device="cuda")
    x[0, 5], x[1, 7], x[2, 9] = float("nan"), float("inf"), -float("inf")
    before = x.clone()
    assert decode.adjust_scores(x, out=x) is x
    assert torch.equal(x.nan_to_num(123.0), before.nan_to_num(123.0))


def test_adjust_masked_places_may_hold_anything():
    """What the grammar forbids is -inf whatever the score, the history or the bias there."""
    for dtype in TYPES.values():
        x = torch.zeros(2, 100, dtype=dtype, device="cuda")
        low = torch.finfo(dtype).min
        x[0, :6] = torch.tensor([float("nan"), float("inf"), -float("inf"), low, 0.0, -0.0])
        x[1, 50:] = low
        ok = np.ones((2, 100), bool)
        ok[0, :6] = False
        ok[1] = False
        bias = torch.zeros(100, device="cuda")
        bias[1], bias[2] = -float("inf"), float("inf")
        tokens = torch.arange(100, dtype=torch.int32, device="cuda").repeat(2, 1)
        got = host(decode.adjust_scores(x, tokens=tokens, repetition=torch.full((2,), 1.3, device="cuda"), bias=bias,
                                        allowed=words_of(ok)))
        assert np.isneginf(got[0, :6]).all() and np.isneginf(got[1]).all()
        assert (got[0, 6:] == 0).all()


def test_adjust_rows_of_a_large_tensor():
    """Rows that start past 2^31 elements."""
    V, N = 1 << 20, 2050
    x = torch.zeros(N, V, dtype=torch.float16, device="cuda")
    x[N - 1] = 1.0
    tokens = torch.full((N, 1), 5, dtype=torch.int32, device="cuda")
    decode.adjust_scores(x, tokens=tokens, presence=torch.full((N,), 3.0, device="cuda"), out=x)
    assert x[N - 1, 5].item() == -2.0 and x[N - 1, 6].item() == 1.0 and x[N - 2, 5].item() == -3.0
    index, _ = decode.choose(x[N - 3:])
    assert index.tolist() == [0, 0, 0]


# ----------------------------------------------------------------------------------- choose
def chosen(z, k, p, min_p, noise):
    """(index, log probability) of one row by the definition; z float64."""
    z = np.where(np.isnan(z), -np.inf, np.minimum(z, np.finfo(np.float32).max))
    order = np.lexsort((np.arange(z.size), -z))
    order = order[z[order] > -np.inf]
    if order.size == 0:
        return -1, -np.inf
    best = z[order[0]]
    if min_p > 0:
        order = order[z[order] >= best + np.log(min_p)]
    if k > 0:
        order = order[:k]
    mass = np.exp(z[order] - best)
    if p < 1:
        before = np.cumsum(mass) - mass
        keep = before < p * mass.sum()
        keep[0] = True
        order, mass = order[keep], mass[keep]
    y = z[order] if noise is None else np.maximum(z[order] + noise[order], -np.finfo(np.float32).max)
    at = order[y == y.max()].min()
    return int(at), float(z[at] - best - np.log(mass.sum()))


def scores_of(kind, N, V, rng):
    """Multiples of 1/8, so that sums and quotients by powers of two are exact and ties are many."""
    if kind == "normal":
        x = np.round(rng.normal(0, 3, (N, V)) * 8) / 8
    elif kind == "peak":
        x = np.round(rng.normal(-8, 1, (N, V)) * 8) / 8
        x[np.arange(N), rng.integers(0, V, N)] = 4.0
    elif kind == "equal":
        x = np.full((N, V), -1.25)
    elif kind == "two":
        x = np.where(rng.random((N, V)) < 0.5, 0.5, -0.5)
    elif kind == "rising":
        x = np.broadcast_to(np.arange(V) * 0.125 - V / 16, (N, V)).copy()
    elif kind == "falling":
        x = np.broadcast_to(-np.arange(V) * 0.125, (N, V)).copy()
    elif kind == "flat":
        x = np.round(rng.random((N, V)) * 2) / 8
    elif kind == "wide":
        x = rng.choice([-1e30, -3e4, -100.0, -0.0, 0.0, 60.0, 60.125], (N, V))
    elif kind == "masked":
        x = np.where(rng.random((N, V)) < 0.97, -np.inf, np.round(rng.normal(0, 3, (N, V)) * 8) / 8)
    elif kind == "none":
        x = np.where(rng.random((N, V)) < 0.1, np.nan, -np.inf)
    else:  # "odd": NaN, infinities, the type's lowest value
        x = np.round(rng.normal(0, 3, (N, V)) * 8) / 8
        x[rng.random((N, V)) < 0.2] = np.nan
        x[rng.random((N, V)) < 0.2] = -np.inf
        x[rng.random((N, V)) < 0.1] = np.finfo(np.float32).min
        x[: N // 2][rng.random((N // 2, V)) < 0.01] = np.inf
    return x.astype(np.float32)


KINDS = ["normal", "peak", "equal", "two", "rising", "falling", "flat", "wide", "masked", "none", "odd"]


def choose_case(N, V, kind, filters, seed, dtype="f32", drawn=True, pad=0, offset=0, temper=True):
    rng = np.random.default_rng(seed)
    with np.errstate(over="ignore"):
        xt = torch.from_numpy(scores_of(kind, N, V, rng)).to(TYPES[dtype]).cuda()
    x = host(xt)
    t = rng.choice([0.5, 1.0, 2.0], N).astype(np.float32) if temper else np.ones(N, np.float32)
    if temper and N > 2:
        t[1] = 0.0
    noise = np.round(-np.log(-np.log(rng.random((N, V)))) * 1024).astype(np.float32) / 1024 if drawn else None
    k = np.zeros(N, np.int32)
    p = np.ones(N, np.float32)
    m = np.zeros(N, np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        z = (x.astype(np.float32) / np.where(t > 0, t, 1)[:, None]).astype(np.float64)
    if "k" in filters:
        k = rng.choice([1, 2, 5, 40, 63, 64, 65, max(1, V // 2), max(1, V - 1), V, V + 5, 0, -3], N).astype(np.int32)
    if "m" in filters:  # between multiples of 1/16, which scores over a temperature of 2 are
        m = np.exp(-(np.round(rng.random(N) * 40) / 8 + 0.03125)).astype(np.float32)
    if "p" in filters:
        for n in range(N):
            row = np.where(np.isnan(z[n]), -np.inf, np.minimum(z[n], np.finfo(np.float32).max))
            order = np.lexsort((np.arange(V), -row))
            order = order[row[order] > -np.inf]
            if order.size == 0:
                continue
            if m[n] > 0:
                order = order[row[order] >= row[order[0]] + np.log(np.float64(m[n]))]
            if k[n] > 0:
                order = order[:k[n]]
            share = np.exp(row[order] - row[order[0]])
            share /= share.sum()
            upto = np.cumsum(share)
            # an end between two answers, neither of which is within the roundings of the other
            able = np.flatnonzero(share > 1e-5)
            if able.size == 0:
                continue
            j = rng.choice(able) if rng.random() < 0.8 else able[-1]
            p[n] = upto[j] - 0.5 * share[j]
    give = lambda on, a: torch.from_numpy(a).cuda() if on else None  # noqa: E731
    nt = None if noise is None else spread(torch.from_numpy(noise).cuda(), pad, offset)
    index, log = decode.choose(spread(xt, pad, offset), temperature=give(temper, t), top_k=give("k" in filters, k),
                               top_p=give("p" in filters, p), min_p=give("m" in filters, m), noise=nt)
    assert index.dtype == torch.int32 and log.dtype == torch.float32
    for n in range(N):
        kk = 1 if t[n] <= 0 else int(k[n])
        want, lp = chosen(z[n], kk, float(p[n]), float(m[n]), None if noise is None else noise[n].astype(np.float64))
        assert index[n].item() == want, (n, kind, filters)
        got = log[n].item()
        # exp within 2 units, sums exact, log within 2 units
        assert got == lp or abs(got - lp) <= 2.0**-20 + 2.0**-22 * abs(lp), (n, got, lp)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("filters", ["", "k", "p", "m", "kp", "km", "mp", "kmp"])
def test_choose_kinds(kind, filters):
    choose_case(13, 3001, kind, filters, 17)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 255, 1000, 1023, 1024, 1025, 4097, 16384, 20001, 70000, 131073])
@pytest.mark.parametrize("filters", ["", "k", "p", "kmp"])
def test_choose_sizes(V, filters):
    for kind in ("normal", "flat", "masked"):
        choose_case(4, V, kind, filters, V)


@pytest.mark.parametrize("kind", ["equal", "two", "flat", "rising", "odd"])
@pytest.mark.parametrize("filters", ["k", "p", "kp"])
def test_choose_large_rows_of_ties(kind, filters):
    """More equal scores than any list of candidates holds."""
    choose_case(5, 50000, kind, filters, 5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("filters", ["", "k", "p", "kmp"])
@pytest.mark.parametrize("drawn", [True, False])
def test_choose_types(dtype, filters, drawn):
    for kind in ("normal", "peak", "odd"):
        choose_case(6, 5003, kind, filters, 3, dtype, drawn)


@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (8, 5)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_choose_strides(pad, offset, dtype):
    choose_case(5, 1501, "normal", "kp", 9, dtype, True, pad, offset)
    choose_case(5, 1501, "normal", "", 9, dtype, True, pad, offset, temper=False)


def test_choose_many_rows():
    choose_case(300, 700, "normal", "kmp", 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["normal", "flat", "odd"])
@pytest.mark.parametrize("filters", ["", "k", "m", "p", "kmp"])
def test_choose_many_long_rows(kind, filters, dtype):
    """Rows long enough to be sliced where they are few, and too many for that."""
    choose_case(66, 66000, kind, filters, 4, dtype)


@pytest.mark.parametrize("dtype,V", [("f32", 32767), ("f32", 32768), ("f16", 65535), ("bf16", 65536), ("f32", 300001)])
@pytest.mark.parametrize("filters", ["", "k", "m", "kmp"])
def test_choose_sliced_rows(dtype, V, filters):
    """Around the length from which few rows are sliced, and slices of the largest size."""
    for kind in ("normal", "masked", "odd"):
        choose_case(3, V, kind, filters, 6, dtype)


def test_choose_filter_ends():
    """Bounds that keep the first answer alone, or all of them."""
    x = torch.tensor([[0.0, 2.0, 1.0, 2.0]], device="cuda").repeat(6, 1)
    p = torch.tensor([0.0, -1.0, 1e-9, 0.4999, 1.0, 2.0], device="cuda")
    noise = torch.tensor([9.0, 0.0, 0.0, 0.5], device="cuda")
    index, log = decode.choose(x, top_p=p, noise=noise)
    assert index.tolist() == [1, 1, 1, 3, 0, 0]
    m = torch.tensor([0.0, 1.0, 0.9, 1e-30, 0.2, 0.5], device="cuda")
    index, log = decode.choose(x, min_p=m, noise=noise)
    assert index.tolist() == [0, 3, 3, 0, 3, 3]
    np.testing.assert_allclose(log[1].item(), np.log(0.5), rtol=2.0**-20)


def test_choose_no_scores():
    index, log = decode.choose(torch.empty(3, 0, device="cuda"))
    assert index.tolist() == [-1] * 3 and bool(torch.isneginf(log).all())
    index, log = decode.choose(torch.empty(0, 10, device="cuda"))
    assert index.shape == (0,) and log.shape == (0,)


def test_choose_draws_from_the_softmax():
    """Shares of many draws, with Gumbel noise, against the probabilities: within 5 deviations."""
    V, N = 40, 60000
    torch.manual_seed(1)
    x = torch.randn(V, device="cuda") * 1.5
    u = torch.rand(N, V, device="cuda", dtype=torch.float64).clamp(1e-12, 1 - 1e-12)
    index, log = decode.choose(x.expand(N, V).contiguous(), noise=(-torch.log(-torch.log(u))).float())
    share = torch.bincount(index.long(), minlength=V).double() / N
    prob = torch.softmax(x.double(), 0)
    assert bool(((share - prob).abs() <= 5 * (prob * (1 - prob) / N).sqrt()).all())
    assert bool((log.double() - prob.log()[index.long()]).abs().max() < 1e-5)


# --------------------------------------------------------------- streams, graphs, refusals
def step(state):
    scores = decode.readout(state["bits"], state["codes"], state["scales"], group=64, clauses=state["C"])
    scores = decode.adjust_scores(scores, tokens=state["tokens"], repetition=state["rep"], allowed=state["ok"])
    return (scores, *decode.choose(scores, temperature=state["t"], top_k=state["k"], top_p=state["p"], noise=state["noise"]))


def step_state(N, C, K, seed):
    rng = np.random.default_rng(seed)
    codes, scales, _ = weights(rng, C, K, 64, "f16", False)
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    return dict(C=C, codes=dev(codes), scales=scales.cuda(), bits=clause_rows(rng, N, C, "bits", True)[0],
                tokens=dev(rng.integers(0, K, (N, 30)).astype(np.int32)), rep=dev(rng.uniform(1, 2, N).astype(np.float32)),
                ok=words_of(rng.random((N, K)) < 0.7), t=dev(rng.uniform(0.5, 1.5, N).astype(np.float32)),
                k=dev(rng.integers(0, 50, N).astype(np.int32)), p=dev(rng.uniform(0.5, 1, N).astype(np.float32)),
                noise=dev(rng.gumbel(size=(N, K)).astype(np.float32)))


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("N,C,K", [(1, 500, 900), (20, 1000, 3000), (70, 640, 2000)])
def test_repeats_and_streams(N, C, K):
    """The same call gives the same bits, whatever ran before and on whatever stream."""
    state = step_state(N, C, K, 1)
    want = step(state)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = [step(state) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(other)
    torch.cuda.synchronize()
    for g in got:
        assert same(want, g)


@pytest.mark.parametrize("N,C,K", [(1, 500, 900), (20, 1000, 40000), (70, 640, 2000)])
def test_captured_into_a_graph(N, C, K):
    """A captured step, replayed over new inputs with other work between the replays."""
    state = step_state(N, C, K, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(state)
    for seed in range(4):
        new = step_state(N, C, K, 10 + seed)
        for name, t in new.items():
            if isinstance(t, torch.Tensor):
                state[name].copy_(t)
        want = step(new)
        for o in out:
            o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(want, out), seed


@pytest.mark.parametrize("N", [1, 9, 20, 64, 100])
@pytest.mark.parametrize("dtype", ["bits", "f16", "f32"])
@pytest.mark.parametrize("C,group", [(40, 32), (200, 32), (200, 128), (1000, 256), (1090, 64)])
def test_infinite_scale(dtype, N, C, group):
    """An infinite scale makes its group's sum infinite, whatever pads the last group."""
    K, groups = 20, -(-C // group)
    codes = torch.full((K, 16 * -(-C // 32)), 0x22, dtype=torch.uint8, device="cuda")  # ones
    scales = torch.ones(K, groups, device="cuda")
    scales[3, groups - 1] = float("inf")
    scales[4, 0] = -float("inf")
    if dtype == "bits":
        x = torch.full((N, -(-C // 32)), -1, dtype=torch.int32, device="cuda")
        got = decode.readout(x, codes, scales, group=group, clauses=C)
    else:
        got = decode.readout(torch.ones(N, C, dtype=TYPES[dtype], device="cuda"), codes, scales, group=group)
    want = torch.full((N, K), float(C), device="cuda")
    want[:, 3], want[:, 4] = float("inf"), -float("inf")
    assert torch.equal(got, want)


def test_one_row_for_all():
    """Rows that are one (stride 0) read as if they were copies."""
    rng = np.random.default_rng(2)
    codes, scales, _ = weights(rng, 300, 40, 32, "f32", True)
    dev = [torch.from_numpy(codes).cuda(), scales.cuda()]
    for N in (5, 40):
        x = torch.randn(1, 300, device="cuda")
        assert torch.equal(decode.readout(x.expand(N, 300), *dev), decode.readout(x.expand(N, 300).contiguous(), *dev))
        s, t = torch.randn(1, 500, device="cuda"), torch.arange(9, dtype=torch.int32, device="cuda").view(1, 9)
        rep, noise = torch.rand(N, device="cuda") + 1, torch.rand(500, device="cuda")
        bias, ok = torch.randn(500, device="cuda"), words_of(rng.random((1, 500)) < 0.8)
        a = decode.adjust_scores(s.expand(N, 500), tokens=t.expand(N, 9), repetition=rep, bias=bias, allowed=ok[0])
        b = decode.adjust_scores(s.expand(N, 500).contiguous(), tokens=t.expand(N, 9).contiguous(), repetition=rep,
                                 bias=bias.expand(N, 500).contiguous(), allowed=ok.expand(N, -1).contiguous())
        assert torch.equal(a, b)
        assert same(decode.choose(s.expand(N, 500), noise=noise, temperature=rep),
                    decode.choose(s.expand(N, 500).contiguous(), noise=noise.expand(N, 500).contiguous(), temperature=rep))


def test_refusals():
    f = lambda *shape, **kw: torch.zeros(*shape, device="cuda", **kw)  # noqa: E731
    i32, u8 = torch.int32, torch.uint8
    x, codes, scales = f(2, 64), f(3, 32, dtype=u8), f(3, 2)
    decode.readout(x, codes, scales)
    wrong = [
        (ValueError, lambda: decode.readout(x[0], codes, scales)),
        (TypeError, lambda: decode.readout(x.double(), codes, scales)),
        (TypeError, lambda: decode.readout(x, codes.int(), scales)),
        (TypeError, lambda: decode.readout(x, codes, scales.double())),
        (TypeError, lambda: decode.readout(x, codes, scales, out=f(2, 3, dtype=i32))),
        (ValueError, lambda: decode.readout(x, codes, scales, group=16)),
        (ValueError, lambda: decode.readout(x, codes, scales, group=64)),
        (ValueError, lambda: decode.readout(x, codes, scales, clauses=63)),
        (ValueError, lambda: decode.readout(f(2, 2, dtype=i32), codes, scales, clauses=65)),
        (ValueError, lambda: decode.readout(x, codes[:, :16], scales)),
        (ValueError, lambda: decode.readout(x, f(3, 40, dtype=u8), scales)),
        (ValueError, lambda: decode.readout(x, f(3, 48, dtype=u8)[:, 8:40], scales)),
        (ValueError, lambda: decode.readout(x, codes, scales[:2])),
        (ValueError, lambda: decode.readout(x, codes, scales, out=f(2, 4))),
        (ValueError, lambda: decode.readout(x.t().contiguous().t(), codes, scales)),
        (ValueError, lambda: decode.readout(x, codes.cpu(), scales)),
        (ValueError, lambda: decode.readout(x.requires_grad_(), codes, scales)),
    ]
    s, t = f(2, 10), f(2, 4, dtype=i32)
    wrong += [
        (TypeError, lambda: decode.adjust_scores(s.int())),
        (TypeError, lambda: decode.adjust_scores(s, tokens=t.long())),
        (ValueError, lambda: decode.adjust_scores(s, tokens=t[:1])),
        (ValueError, lambda: decode.adjust_scores(s, lengths=f(2, dtype=i32))),
        (ValueError, lambda: decode.adjust_scores(s, repetition=f(2))),
        (TypeError, lambda: decode.adjust_scores(s, tokens=t, lengths=f(2))),
        (ValueError, lambda: decode.adjust_scores(s, tokens=t, lengths=f(3, dtype=i32))),
        (TypeError, lambda: decode.adjust_scores(s, tokens=t, frequency=f(2, dtype=torch.float16))),
        (ValueError, lambda: decode.adjust_scores(s, bias=f(9))),
        (ValueError, lambda: decode.adjust_scores(s, bias=f(1, 10))),
        (TypeError, lambda: decode.adjust_scores(s, bias=f(10, dtype=torch.float16))),
        (ValueError, lambda: decode.adjust_scores(s, allowed=f(2, 2, dtype=i32))),
        (TypeError, lambda: decode.adjust_scores(s, allowed=f(2, 1))),
        (ValueError, lambda: decode.adjust_scores(s, out=f(2, 9))),
        (TypeError, lambda: decode.adjust_scores(s, out=f(2, 10, dtype=torch.float64))),
        (ValueError, lambda: decode.adjust_scores(s.t())),
        (ValueError, lambda: decode.choose(s[0])),
        (TypeError, lambda: decode.choose(s.double())),
        (TypeError, lambda: decode.choose(s, temperature=1.0)),
        (ValueError, lambda: decode.choose(s, temperature=f(3))),
        (TypeError, lambda: decode.choose(s, top_k=f(2))),
        (TypeError, lambda: decode.choose(s, top_p=f(2, dtype=torch.float64))),
        (ValueError, lambda: decode.choose(s, min_p=f(1))),
        (ValueError, lambda: decode.choose(s, noise=f(2, 9))),
        (TypeError, lambda: decode.choose(s, noise=f(2, 10, dtype=torch.float16))),
        (ValueError, lambda: decode.choose(s.requires_grad_())),
    ]
    for n, (error, call) in enumerate(wrong):
        with pytest.raises(error):
            call()
            print("not refused:", n)
    with torch.no_grad():
        decode.choose(s)
