"""The adapting and learning operators on the GPU against plain numpy in 64 bits.

Where every product and sum is a whole number that float32 holds, results have to be equal.  Elsewhere the
bounds are those of the roundings made: a float32 sum of n terms is within n 2^-23 sum |terms| (twice the
bound of rounding to nearest, for an adder that cuts), an output of 8 or 11 bits of fraction within half of
its last one.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ytm_amd = pytest.importorskip("ytm_amd")
from ytm_amd import decode, tune  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a unit in the last place, relative, and the least difference of numbers near zero
ROUND = {"f32": (2.0**-24, 2.0**-149), "f16": (2.0**-11, 2.0**-25), "bf16": (2.0**-8, 2.0**-133)}


def host(t):
    return t.detach().double().cpu().numpy()


def gpu(v, kind="f32"):
    return torch.from_numpy(np.asarray(v, np.float32)).to(TYPES[kind]).cuda()


def ints(v):
    return torch.from_numpy(np.asarray(v, np.int32)).cuda()


def spread(t, pad, offset=0):
    """The same tensor with its rows `pad` elements further apart, off by `offset`, 77 between them."""
    *front, width = t.shape
    rows = int(np.prod(front))
    big = torch.full((rows * (width + pad) + offset,), 77, dtype=t.dtype, device=t.device)
    out = big[offset:].view(*front, width + pad)[..., :width]
    out.copy_(t)
    return out


def untouched(t, pad, offset=0):
    """Whether what lies between the rows of a spread tensor is still 77."""
    rows, width = int(np.prod(t.shape[:-1])), t.shape[-1]
    whole = t.as_strided((rows, width + pad), (width + pad, 1), offset)
    return bool((whole[:, width:] == 77).all())


# ------------------------------------------------------------------------------- adapters
def clause_rows(rng, N, C, x, exact):
    """(tensor, its values)"""
    if x == "bits":
        on = (rng.random((N, C)) < 0.3).astype(np.uint32)
        words = decode.pack_outputs(on)
        if C % 32:  # bits past the last clause are ignored
            words[:, -1] |= -(1 << C % 32)
        return words, on.astype(np.float64)
    v = rng.integers(-2, 3, (N, C)) if exact else rng.normal(0, 1, (N, C))
    t = gpu(v, x)
    return t, host(t)


class Case:
    """Operands of adapt, their values, and what comes out in 64 bits."""

    def __init__(self, N, C, K, r, M, x="bits", w="f32", scores="f32", exact=True, seed=0, which=None):
        rng = np.random.default_rng([N, C, K, r, M, seed])
        self.N, self.C, self.K, self.r, self.M, self.scale = N, C, K, r, M, 0.5
        self.x, self.xv = clause_rows(rng, N, C, x, exact)
        small = (lambda *s: rng.integers(-1, 2, s)) if exact else (lambda *s: rng.normal(0, 1, s))
        self.down, self.up = gpu(small(M, r, C), w), gpu(small(M, K, r), w)
        self.scores = gpu(rng.integers(-4, 5, (N, K)) if exact else rng.normal(0, 3, (N, K)), scores)
        # some rows without an adapter, said in different ways
        numbers = rng.integers(0, M, N) if M else np.zeros(N, int)
        numbers = np.where(rng.random(N) < 0.15, rng.choice([-1, M, M + 7, -2**31, 2**31 - 1], N), numbers)
        self.which = ints(numbers if which is None else which)
        self.numbers = host(self.which).astype(np.int64)
        self.named = (self.numbers >= 0) & (self.numbers < M)
        d, u = host(self.down), host(self.up)
        self.hidden, self.hidden_size = np.zeros((N, r)), np.zeros((N, r))
        self.out, self.out_size = host(self.scores), np.abs(host(self.scores))
        for n in np.flatnonzero(self.named):
            a = self.numbers[n]
            self.hidden[n], self.hidden_size[n] = d[a] @ self.xv[n], np.abs(d[a]) @ np.abs(self.xv[n])
            self.out[n] += self.scale * (u[a] @ self.hidden[n])
            self.out_size[n] += self.scale * (np.abs(u[a]) @ self.hidden_size[n])

    def adapt(self, **kw):
        kw.setdefault("hidden", torch.full((self.N, self.r), 77.0, device="cuda"))
        return decode_first(tune.adapt(self.scores, self.x, self.down, self.up, self.which, self.scale, **kw), kw)

    def gradients(self, grad, hidden):
        """d_down, d_up of grad (N, K) and hidden (N, r), and the same of their sizes."""
        u = host(self.up)
        back, size = np.zeros((self.N, self.r)), np.zeros((self.N, self.r))
        for n in np.flatnonzero(self.named):
            back[n] = self.scale * (grad[n] @ u[self.numbers[n]])
            size[n] = self.scale * (np.abs(grad[n]) @ np.abs(u[self.numbers[n]]))
        found = []
        for g, b, h, x in ((grad, back, hidden, self.xv), (np.abs(grad), size, np.abs(hidden), np.abs(self.xv))):
            d_down, d_up = np.zeros((self.M, self.r, self.C)), np.zeros((self.M, self.K, self.r))
            for a in range(self.M):
                rows = self.named & (self.numbers == a)
                d_down[a], d_up[a] = b[rows].T @ x[rows], self.scale * (g[rows].T @ h[rows])
            found.append((d_down, d_up))
        return found


def decode_first(out, kw):
    return out, kw["hidden"]


SIZES = [(1, 1, 1, 1, 1), (1, 2000, 10, 8, 4), (2, 33, 17, 5, 3), (3, 31, 5, 3, 1), (15, 64, 15, 16, 2),
         (16, 128, 64, 16, 1), (17, 129, 65, 17, 5), (48, 1000, 300, 16, 40), (64, 257, 130, 33, 64),
         (100, 96, 70, 64, 7), (256, 300, 40, 4, 9), (257, 300, 40, 4, 9), (600, 70, 33, 8, 3), (40, 500, 1000, 130, 2),
         (5, 4097, 513, 2, 300), (1500, 65, 20, 1, 700), (8, 100, 50, 256, 2)]


@pytest.mark.parametrize("x,w", [("bits", "f32"), ("bits", "f16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"),
                                 ("f32", "bf16"), ("f16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("N,C,K,r,M", SIZES)
def test_adapt_exact(N, C, K, r, M, x, w):
    """Small whole numbers: every sum is exact."""
    c = Case(N, C, K, r, M, x, w)
    out, hidden = c.adapt()
    np.testing.assert_array_equal(host(hidden), c.hidden)
    np.testing.assert_array_equal(host(out), c.out)


@pytest.mark.parametrize("x,w", [("bits", "f32"), ("bits", "bf16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"),
                                 ("f32", "f16")])
@pytest.mark.parametrize("N,C,K,r,M", SIZES)
def test_gradient_exact(N, C, K, r, M, x, w):
    c = Case(N, C, K, r, M, x, w)
    rng = np.random.default_rng(1)
    grad, hidden = rng.integers(-1, 2, (N, K)), rng.integers(-2, 3, (N, r))
    # of 16-bit outputs: sums that their fraction holds
    kind = "f32" if w == "f32" else w
    (d_down, d_up), _ = c.gradients(grad.astype(float), hidden.astype(float))
    got = tune.adapt_gradient(gpu(grad), c.x, c.down, c.up, c.which, gpu(hidden), c.scale)
    for g, want in zip(got, (d_down, d_up)):
        rounded = host(torch.from_numpy(want).float().to(TYPES[kind]))  # float32 holds the sums
        np.testing.assert_array_equal(host(g), rounded)


def within(got, want, size, terms, out):
    rel, least = ROUND[out]
    err = np.abs(host(got) - want)
    bound = terms * 2.0**-23 * size + rel * np.abs(want) + least
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("x,w,scores,out", [("bits", "f32", "f32", "f32"), ("bits", "f16", "f16", "bf16"),
                                            ("f32", "f32", "bf16", "f16"), ("f16", "f16", "f32", "f32"),
                                            ("bf16", "bf16", "bf16", "bf16"), ("f32", "bf16", "f16", "f32")])
@pytest.mark.parametrize("N,C,K,r,M", [(1, 500, 40, 4, 1), (40, 777, 129, 16, 9), (300, 333, 65, 40, 4)])
def test_adapt_types(N, C, K, r, M, x, w, scores, out):
    c = Case(N, C, K, r, M, x, w, scores, exact=False)
    to = torch.empty(N, K, dtype=TYPES[out], device="cuda")
    got, hidden = c.adapt(out=to)
    assert got is to
    within(hidden, c.hidden, c.hidden_size, C, "f32")
    within(got, c.out, c.out_size, C + r + 1, out)


@pytest.mark.parametrize("x,w,kind", [("bits", "f32", "f32"), ("bits", "f16", "f32"), ("f32", "f32", "bf16"),
                                      ("f16", "f16", "f16"), ("bf16", "bf16", "bf16"), ("f32", "bf16", "f16")])
@pytest.mark.parametrize("N,C,K,r,M", [(1, 500, 40, 4, 1), (40, 777, 129, 16, 9), (300, 333, 65, 40, 4)])
def test_gradient_types(N, C, K, r, M, x, w, kind):
    c = Case(N, C, K, r, M, x, w, exact=False)
    rng = np.random.default_rng(2)
    grad, hidden = gpu(rng.normal(0, 1, (N, K)), kind), gpu(rng.normal(0, 1, (N, r)))
    want, size = c.gradients(host(grad), host(hidden))
    got = tune.adapt_gradient(grad, c.x, c.down, c.up, c.which, hidden, c.scale)
    within(got[0], want[0], size[0], N + K + 1, w)
    within(got[1], want[1], size[1], N + 1, w)


def test_gradient_against_differences():
    """A loss sum(out * g): with whole numbers its differences along a coordinate are exact."""
    c = Case(9, 50, 30, 5, 3, "bits")
    rng = np.random.default_rng(5)
    g = gpu(rng.integers(-2, 3, (9, 30)))
    out, hidden = c.adapt()
    d_down, d_up = tune.adapt_gradient(g, c.x, c.down, c.up, c.which, hidden, c.scale)
    base = (host(out) * host(g)).sum()
    for t, d in ((c.down, d_down), (c.up, d_up)):
        for _ in range(12):
            at = tuple(int(rng.integers(0, s)) for s in t.shape)
            t[at] += 1.0
            moved, _ = c.adapt()
            assert (host(moved) * host(g)).sum() - base == float(d[at])
            t[at] -= 1.0


@pytest.mark.parametrize("N", [5, 40, 300])
@pytest.mark.parametrize("x,pad,offset", [("bits", 2, 1), ("f32", 3, 1), ("f16", 5, 1), ("bf16", 8, 8)])
def test_adapt_strides(x, pad, offset, N):
    w = "f32" if x == "bits" else x
    c = Case(N, 133, 70, 6, 4, x, w)
    hidden = spread(torch.zeros(N, 6, device="cuda"), 3, 2)
    to = spread(torch.zeros(N, 70, device="cuda"), 5, 3)
    down, up = spread(c.down, pad, offset), spread(c.up, pad, offset)
    got = tune.adapt(spread(c.scores, 1, 1), spread(c.x, pad, offset), down, up, c.which, c.scale, hidden=hidden, out=to)
    np.testing.assert_array_equal(host(hidden), c.hidden)
    np.testing.assert_array_equal(host(got), c.out)
    assert untouched(hidden, 3, 2) and untouched(to, 5, 3)
    grad = np.random.default_rng(3).integers(-1, 2, (N, 70)).astype(float)
    (d_down, d_up), _ = c.gradients(grad, c.hidden)
    to = spread(torch.zeros_like(c.down), pad, offset), spread(torch.zeros_like(c.up), 1, offset)
    got = tune.adapt_gradient(spread(gpu(grad), pad, offset), spread(c.x, pad, offset), down, up, c.which, hidden,
                              c.scale, out=to)
    assert got[0] is to[0] and got[1] is to[1]
    for t, want, p in zip(to, (d_down, d_up), (pad, 1)):
        np.testing.assert_array_equal(host(t), host(torch.from_numpy(want).float().to(TYPES[w])))
        assert untouched(t, p, offset)


def test_adapt_in_place_and_one_for_all():
    c = Case(33, 100, 90, 7, 3)
    want = c.out
    scores = c.scores.clone()
    assert tune.adapt(scores, c.x, c.down, c.up, c.which, c.scale, out=scores) is scores
    np.testing.assert_array_equal(host(scores), want)
    # one adapter's memory for all, one row's scores for all
    one = Case(33, 100, 90, 7, 1, which=np.zeros(33))
    down, up = one.down.expand(3, -1, -1), one.up.expand(3, -1, -1)
    which = ints(np.arange(33) % 3)
    got = tune.adapt(one.scores[:1].expand(33, -1), one.x, down, up, which, one.scale)
    np.testing.assert_array_equal(host(got), one.out - host(one.scores) + host(one.scores[:1]))


def test_adapters_in_one_buffer():
    """down and up of each adapter one after the other in memory: gradients go there too."""
    M, r, C, K, N = 4, 3, 50, 20, 60
    c = Case(N, C, K, r, M)
    each = r * C + K * r
    def views(flat):
        return (flat.as_strided((M, r, C), (each, C, 1)), flat.as_strided((M, K, r), (each, r, 1), r * C))
    flat, grads = torch.zeros(M * each, device="cuda"), torch.full((M * each,), 77.0, device="cuda")
    down, up = views(flat)
    down.copy_(c.down)
    up.copy_(c.up)
    hidden = torch.empty(N, r, device="cuda")
    got = tune.adapt(c.scores, c.x, down, up, c.which, c.scale, hidden=hidden)
    np.testing.assert_array_equal(host(got), c.out)
    grad = np.random.default_rng(3).integers(-1, 2, (N, K)).astype(float)
    want, _ = c.gradients(grad, c.hidden)
    d_down, d_up = tune.adapt_gradient(gpu(grad), c.x, down, up, c.which, hidden, c.scale, out=views(grads))
    np.testing.assert_array_equal(host(d_down), want[0])
    np.testing.assert_array_equal(host(d_up), want[1])


@pytest.mark.parametrize("N,C,K,M", [(0, 50, 20, 2), (7, 0, 20, 2), (7, 50, 0, 2), (7, 50, 20, 0)])
def test_adapt_nothing(N, C, K, M):
    c = Case(N, C, K, 3, M)
    out, hidden = c.adapt()
    np.testing.assert_array_equal(host(out), c.out)
    np.testing.assert_array_equal(host(hidden), c.hidden)
    grad = np.ones((N, K))
    (d_down, d_up), _ = c.gradients(grad, c.hidden)
    got = tune.adapt_gradient(gpu(grad), c.x, c.down, c.up, c.which, hidden, c.scale)
    np.testing.assert_array_equal(host(got[0]), d_down)
    np.testing.assert_array_equal(host(got[1]), d_up)


@pytest.mark.parametrize("N", [20, 300])
def test_adapt_infinities_stay_in_their_rows_and_adapters(N):
    c = Case(N, 70, 40, 6, 5, "f32", which=np.arange(N) % 5)
    bad = c.numbers == 2
    c.x[np.flatnonzero(c.numbers == 1)[0], 3] = float("inf")
    row = int(np.flatnonzero(c.numbers == 1)[0])
    c.up[2, 4, 1] = float("nan")
    c.down[3, 2, 5] = float("inf")
    out, hidden = c.adapt()
    out, hidden = host(out), host(hidden)
    clean = ~bad & (c.numbers != 3)
    clean[row] = False
    np.testing.assert_array_equal(out[clean], c.out[clean])
    assert np.isnan(out[bad][:, 4]).all()
    np.testing.assert_array_equal(np.delete(out[bad], 4, 1), np.delete(c.out[bad], 4, 1))
    assert not np.isfinite(hidden[row]).all()
    np.testing.assert_array_equal(np.delete(hidden[c.numbers == 3], 2, 1), np.delete(c.hidden[c.numbers == 3], 2, 1))
    # a gradient that is not finite reaches its own adapter's and no other's
    grad = np.random.default_rng(3).integers(-1, 2, (N, 40)).astype(float)
    c = Case(N, 70, 40, 6, 5, "f32", which=np.arange(N) % 5)
    want, _ = c.gradients(grad, c.hidden)
    g = gpu(grad)
    g[int(np.flatnonzero(c.numbers == 1)[0]), 7] = float("nan")
    got = [host(t) for t in tune.adapt_gradient(g, c.x, c.down, c.up, c.which, gpu(c.hidden), c.scale)]
    for a in range(5):
        for t, w in zip(got, want):
            if a == 1:
                assert np.isnan(t[a]).any()
            else:
                np.testing.assert_array_equal(t[a], w[a])
    np.testing.assert_array_equal(np.delete(got[1][1], 7, 0), np.delete(want[1][1], 7, 0))


def test_adapter_past_32_bits():
    """The last of adapters whose elements 32 bits do not count."""
    M, r, C, K = 3, 256, 5, 8
    apart = 1 << 30  # elements, 2 GiB of float16
    flat = torch.zeros(2 * apart + max(r * C, K * r), dtype=torch.float16, device="cuda")
    c = Case(20, C, K, r, M, "bits", "f16")
    down = flat.as_strided((M, r, C), (apart, C, 1))
    down.copy_(c.down)
    np.testing.assert_array_equal(host(tune.adapt(c.scores, c.x, down, c.up, c.which, c.scale)), c.out)
    grad = np.random.default_rng(3).integers(-1, 2, (20, K)).astype(float)
    want, _ = c.gradients(grad, c.hidden)
    up = flat.as_strided((M, K, r), (apart, r, 1))
    got = tune.adapt_gradient(gpu(grad), c.x, c.down, c.up, c.which, gpu(c.hidden), c.scale,
                              out=(torch.empty_like(c.down), up))
    np.testing.assert_array_equal(host(got[1]), host(torch.from_numpy(want[1]).to(torch.float16)))


@pytest.mark.parametrize("N,M", [(65535, 4), (20000, 3000), (300, 65535)])
def test_adapt_many_rows_and_adapters(N, M):
    c = Case(N, 37, 5, 2, M)
    out, hidden = c.adapt()
    np.testing.assert_array_equal(host(hidden), c.hidden)
    np.testing.assert_array_equal(host(out), c.out)
    rng = np.random.default_rng(1)
    grad, h = rng.integers(-1, 2, (N, 5)), rng.integers(-1, 2, (N, 2))
    rows = np.flatnonzero(c.named)
    at, u, xv = c.numbers[rows], host(c.up), c.xv[rows]
    back = c.scale * np.einsum("no,noj->nj", grad[rows].astype(float), u[at])
    d_down, d_up = np.zeros((M, 2, 37)), np.zeros((M, 5, 2))
    np.add.at(d_down, at, back[:, :, None] * xv[:, None, :])
    np.add.at(d_up, at, c.scale * grad[rows][:, :, None] * h[rows][:, None, :])
    got = tune.adapt_gradient(gpu(grad), c.x, c.down, c.up, c.which, gpu(h), c.scale)
    np.testing.assert_array_equal(host(got[0]), d_down)
    np.testing.assert_array_equal(host(got[1]), d_up)


# --------------------------------------------------------------------------------- losses
def score_rows(rng, N, V, kind, masked=0.2):
    s = rng.normal(0, 3, (N, V)).astype(np.float32)
    s[rng.random((N, V)) < masked] = -np.inf
    return gpu(s, kind)


def log_softmax(scores, temperature):
    """log softmax (N, V) of the values the operators take, and the bound of a float32 log probability's error."""
    z = np.where(np.isnan(scores), -np.inf, np.minimum(scores, np.finfo(np.float32).max))
    t = np.ones(len(z)) if temperature is None else np.asarray(temperature, np.float64)
    heat = np.where(t <= 0, 1.0, np.where(t >= 2.0**-126, t, 2.0**-126))
    z = z / heat[:, None]
    with np.errstate(invalid="ignore", divide="ignore"):
        best = z.max(1, keepdims=True, initial=-np.inf)
        e = np.where(z > -np.inf, np.exp(z - best), 0.0)
        total = e.sum(1, keepdims=True)
        log = z - best - np.log(total)
        p = np.where(e > 0, e / total, 0.0)
    # a term's exponent d = z - best is rounded three times (difference, factor, product), its power to 2 units; the
    # mean of d over p is at most log V + 1.  Sums: V terms in chains of at most V / 64 + 64.
    V = z.shape[1]
    return log, p, heat, 2.0**-23 * (3 * (np.log(max(V, 2)) + 1) + 4) + 2.0**-24 * (V / 64 + 64 + 16)


def check_grad(got, scores, tokens, p, c, c_err, heat, eps, out):
    """grad = c / heat * (onehot - p), c off by at most c_err, p by a share of what its exponent's rounding and eps
    give."""
    N, V = scores.shape
    one = np.zeros((N, V))
    rows = np.flatnonzero(c != 0)
    one[rows, tokens[rows]] = 1.0
    want = (c / heat)[:, None] * (one - p)
    want[c == 0] = 0.0
    with np.errstate(divide="ignore"):
        far = np.where(p > 0, -np.log(np.where(p > 0, p, 1.0)), 0.0) + np.log(V + 1.0)
    size = (one + p) * (np.abs(c) / heat)[:, None]
    rel, least = ROUND[out]
    bound = (one + p) * (c_err / heat)[:, None] + size * (eps + 2.0**-22 * (far + 4)) + rel * np.abs(want) * 1.01 + least
    # a power below the least normal number, 2^-126, is 0; it is divided by a sum of powers that is above 2^-24 2^-0.5 (one
    # relative to a whole exponent near a score, taken where it is above 2^-24, or to the largest score itself)
    bound += (np.abs(c) / heat)[:, None] * 2.0**(-126 + 24.5)
    err = np.abs(host(got) - want)
    err[np.isnan(err)] = np.inf
    assert (err <= bound).all(), (err / bound).max()


def policy_want(log, tokens, old, adv, ref, kl, low, high, w):
    N, V = log.shape
    there = (tokens >= 0) & (tokens < V)
    lp = np.where(there, log[np.arange(N), np.clip(tokens, 0, V - 1)], -np.inf)
    there &= lp > -np.inf
    lp = np.where(there, lp, 0.0)
    ratio = np.exp(lp - old)
    free, held = ratio * adv, np.clip(ratio, 1 - low, 1 + high) * adv
    loss, c, size = -np.minimum(free, held), -np.where(free <= held, free, 0.0), np.abs(free) + np.abs(held)
    if kl:
        far = ref - lp
        loss, c = loss + kl * (np.expm1(far) - far), c - kl * np.expm1(far)
        size = size + kl * (np.exp(far) + np.abs(far) + 1)
    return tuple(np.where(there, v, 0.0) for v in (w * loss, w * c, w * size, lp))


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("N", [5, 600])
def test_policy_scores_far_from_zero(N, kind):
    """Whole rows at the ends of a type, masked beginnings of rows, temperatures of all sizes."""
    rng = np.random.default_rng(N)
    V, end = 3000, 6e4 if kind == "f16" else 3e38
    s = rng.normal(0, 3, (N, V)).astype(np.float32)
    s[0] = s[0] * 1e-3 - 200.0
    s[1] = s[1] * 1e-3 + 300.0
    s[2] = np.where(rng.random(V) < 0.5, end, -end)
    s[3, :2900] = -np.inf
    s[4, ::8] = -1e4  # each thread's first scores far below the others
    temperature = np.ones(N, np.float32)
    temperature[5:] = 10.0 ** rng.uniform(-3, 3, N - 5)
    scores = gpu(s, kind)
    log, p, heat, eps = log_softmax(host(scores), temperature)
    tokens = np.where(np.arange(N) == 3, 2950, host(scores).argmax(1))
    want = log[np.arange(N), tokens]
    old = want.astype(np.float32)
    losses, grad, lp = tune.policy_loss(scores, ints(tokens), gpu(old), gpu(np.full(N, 1.0)), weights=gpu(np.ones(N)),
                                        temperature=gpu(temperature))
    lp_err = eps + 2.0**-24 * np.abs(want) + 2.0**-22
    assert (np.abs(host(lp) - want) <= lp_err).all()
    check_grad(grad, host(scores), tokens, p, np.full(N, -1.0), np.full(N, 1.0) * (1.1 * lp_err + 2.0**-21), heat, eps, "f32")


VOCABULARIES = [(1, 1), (5, 2), (3, 10), (7, 63), (4, 64), (300, 65), (2, 1000), (33, 4097), (1, 10000), (6, 32001),
                (2, 131072), (600, 8192)]


@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("N,V", VOCABULARIES)
@pytest.mark.parametrize("full", [False, True])
def test_policy(N, V, kind, out, full):
    rng = np.random.default_rng([N, V, full])
    scores = score_rows(rng, N, V, kind)
    temperature = rng.uniform(0.3, 2.0, N).astype(np.float32) if full else None
    if full and N > 3:
        temperature[1], temperature[2] = 0.0, -1.0
    log, p, heat, eps = log_softmax(host(scores), temperature)
    tokens = rng.integers(0, V, N)
    tokens[rng.random(N) < 0.2] = rng.choice([-1, V, 2**31 - 1])
    lp = log[np.arange(N), np.clip(tokens, 0, V - 1)]
    lp[~np.isfinite(lp)] = -5.0
    # ratios away from the clip's bounds, at which the gradient jumps
    old = (lp - np.log(rng.choice([0.4, 0.7, 0.9, 1.0, 1.1, 1.4, 3.0], N))).astype(np.float32)
    adv = rng.normal(0, 1, N).astype(np.float32)
    ref = (lp + rng.normal(0, 0.5, N)).astype(np.float32)
    w = rng.uniform(0.1, 1.0, N).astype(np.float32) if full else np.full(N, np.float32(1) / np.float32(N))
    kl, low, high = (0.25, 0.2, 0.3) if full else (0.0, 0.2, 0.2)
    want = policy_want(log, tokens, old.astype(float), adv.astype(float), ref.astype(float), kl, low, high, w.astype(float))
    to = torch.full((N, V), 77.0, dtype=TYPES[out], device="cuda")
    losses, grad, logprobs = tune.policy_loss(
        scores, ints(tokens), gpu(old), gpu(adv), reference=gpu(ref) if full else None, kl=kl, clip=low,
        clip_high=high if full else None, weights=gpu(w) if full else None,
        temperature=gpu(temperature) if full else None, out=to)
    assert grad is to
    # a log probability: eps of its sum, then half a unit of itself; of it a ratio's error, and a few units more
    lp_err = eps + 2.0**-24 * np.abs(want[3]) + 2.0**-22
    assert (np.abs(host(logprobs) - want[3]) <= lp_err).all()
    c_err = want[2] * (1.1 * lp_err + 2.0**-21)
    assert (np.abs(host(losses) - want[0]) <= c_err).all()
    check_grad(grad, host(scores), tokens, p, want[1], c_err, heat, eps, out)


def preference_want(log, tokens, starts, ref, beta, smoothing):
    N, V = log.shape
    there = (tokens >= 0) & (tokens < V)
    lp = np.where(there, log[np.arange(N), np.clip(tokens, 0, V - 1)], -np.inf)
    there &= lp > -np.inf
    lp = np.where(there, lp, 0.0)
    pairs = len(ref) // 2
    said = np.array([lp[a:max(a, b)].sum() for a, b in zip(starts[:-1], starts[1:])])
    m = beta * ((said - ref)[0::2] - (said - ref)[1::2])
    losses = ((1 - smoothing) * np.logaddexp(0, -m) + smoothing * np.logaddexp(0, m)) / pairs
    slope = beta * (smoothing / (1 + np.exp(-m)) - (1 - smoothing) / (1 + np.exp(m))) / pairs
    c = np.zeros(N)
    for s in range(2 * pairs):
        c[starts[s]:starts[s + 1]] = slope[s // 2] * (1 if s % 2 == 0 else -1)
    return losses, np.where(there, c, 0.0), said, lp, m


@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("N,V,pairs", [(2, 2, 1), (7, 10, 1), (40, 65, 5), (300, 1000, 7), (33, 4097, 16), (5, 32001, 1),
                                       (700, 300, 200), (3, 131072, 1), (1, 50, 4)])
@pytest.mark.parametrize("full", [False, True])
def test_preference(N, V, pairs, kind, out, full):
    rng = np.random.default_rng([N, V, pairs, full])
    scores = score_rows(rng, N, V, kind)
    temperature = rng.uniform(0.3, 2.0, N).astype(np.float32) if full else None
    log, p, heat, eps = log_softmax(host(scores), temperature)
    tokens = rng.integers(0, V, N)
    tokens[rng.random(N) < 0.1] = -1
    used = N - N // 8 if full else N  # some rows before the first and behind the last sequence
    starts = np.sort(np.concatenate(([used // 10 if full else 0, used], rng.integers(used // 10 if full else 0, used + 1, 2 * pairs - 1))))
    beta, smoothing = (0.3, 0.1) if full else (0.1, 0.0)
    none = preference_want(log, tokens, starts, np.zeros(2 * pairs), beta, smoothing)
    ref = (none[2] + rng.normal(0, 5, 2 * pairs)).astype(np.float32)
    want = preference_want(log, tokens, starts, ref.astype(float), beta, smoothing)
    to = torch.full((N, V), 77.0, dtype=TYPES[out], device="cuda")
    losses, grad, said = tune.preference_loss(scores, ints(tokens), ints(starts), gpu(ref), beta=beta, smoothing=smoothing,
                                              temperature=gpu(temperature) if full else None, out=to)
    assert grad is to
    lp_err = np.concatenate(([0.0], np.cumsum(eps + 2.0**-24 * np.abs(want[3]) + 2.0**-22)))
    said_err = lp_err[starts[1:]] - lp_err[starts[:-1]]
    assert (np.abs(host(said) - want[2]) <= said_err + 2.0**-24 * np.abs(want[2])).all()
    m_err = beta * (said_err[0::2] + said_err[1::2]) * 1.01 + 2.0**-23 * np.abs(want[4])
    # both parts of a loss grow by at most m_err; powers and logarithms of float32 to 4 units
    assert (np.abs(host(losses) - want[0]) <= (m_err + 2.0**-21 * (1 + np.abs(want[4]))) / pairs).all()
    c_err = np.zeros(N)
    for s in range(2 * pairs):
        c_err[starts[s]:starts[s + 1]] = beta / pairs * (m_err[s // 2] + 2.0**-21)
    check_grad(grad, host(scores), tokens, p, want[1], np.where(want[1] != 0, c_err, 0.0), heat, eps, out)


@pytest.mark.parametrize("V", [40, 5000, 70000])
def test_losses_rows_that_a_mask_leaves_empty(V):
    """Rows of -inf or NaN alone, answers that a mask leaves out, infinities beside answers."""
    rng = np.random.default_rng(V)
    N = 8
    s = rng.normal(0, 2, (N, V)).astype(np.float32)
    tokens = rng.integers(1, V - 1, N)
    s[0] = -np.inf
    s[1] = np.nan
    s[2, tokens[2]] = -np.inf
    s[3, tokens[3]] = np.nan
    s[4, 0], s[4, V - 1] = np.nan, -np.inf
    s[5, 0] = np.inf  # all of the mass
    s[6] = np.finfo(np.float32).min  # the type's lowest value is no -inf
    s[7, tokens[7]] = np.inf
    with np.errstate(over="ignore"):
        log, p, heat, eps = log_softmax(s.astype(np.float64), None)
    old, adv = np.full(N, -3.0, np.float32), np.linspace(0.5, 2, N).astype(np.float32)
    lp = log[np.arange(N), tokens]
    old = np.where(np.isfinite(lp), np.clip(lp, -50, 0) - 0.05, -3).astype(np.float32)
    losses, grad, logprobs = tune.policy_loss(gpu(s), ints(tokens), gpu(old), gpu(adv))
    assert bool((grad[:4] == 0).all()) and bool((losses[:4] == 0).all()) and bool((logprobs[:4] == 0).all())
    assert bool(torch.isfinite(grad).all()) and bool(torch.isfinite(losses).all())
    assert float(grad[4, 0]) == 0 and float(grad[4, V - 1]) == 0
    assert abs(float(logprobs[6]) + np.log(V)) <= eps + 2.0**-20
    assert float(logprobs[7]) == 0.0 and bool((grad[7] == 0).all())  # certain: nothing to gain
    starts = ints([0, 4, 8])
    losses, grad, said = tune.preference_loss(gpu(s), ints(tokens), starts, gpu([0.0, -100.0]))
    assert float(said[0]) == 0.0 and bool((grad[:4] == 0).all())
    ok = [4, 6, 7]
    assert bool(torch.isfinite(grad[ok]).all())


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,V", [(5, 1003), (3, 40001), (200, 4097)])
def test_losses_in_place_and_strides(N, V, kind):
    rng = np.random.default_rng(N)
    scores = score_rows(rng, N, V, kind)
    tokens, old, adv = ints(rng.integers(0, V, N)), gpu(np.full(N, -4.0)), gpu(rng.normal(0, 1, N))
    to = torch.empty(N, V, dtype=TYPES[kind], device="cuda")
    a = tune.policy_loss(scores, tokens, old, adv, out=to)
    wide = spread(scores, 5, 3)
    far = spread(torch.zeros_like(scores), 2, 1)
    b = tune.policy_loss(wide, tokens, old, adv, out=far)
    own = scores.clone()
    c = tune.policy_loss(own, tokens, old, adv, out=own)
    assert c[1] is own and untouched(far, 2, 1) and untouched(wide, 5, 3)
    for q in (b, c):
        for s, t in zip(a, q):
            assert torch.equal(s, t)
    starts, ref = ints([0, N // 2, N - 1]), gpu([-3.0, -4.0])
    a = tune.preference_loss(scores, tokens, starts, ref, out=to.clone())
    far = spread(torch.zeros_like(scores), 2, 1)
    b = tune.preference_loss(wide, tokens, starts, ref, out=far)
    own = scores.clone()
    c = tune.preference_loss(own, tokens, starts, ref, out=own)
    assert untouched(far, 2, 1) and untouched(wide, 5, 3) and bool((a[1][N - 1:] == 0).all())
    for q in (b, c):
        for s, t in zip(a, q):
            assert torch.equal(s, t)


def test_losses_past_32_bits():
    """The last rows of scores whose elements 32 bits do not count, in place."""
    N, V, last = 17000, 131072, 3
    rng = np.random.default_rng(0)
    s = score_rows(rng, last, V, "bf16")
    tokens = np.full(N, -1)
    tokens[-last:] = rng.integers(0, V, last)
    s[torch.arange(last), torch.from_numpy(tokens[-last:]).cuda()] = 1.0
    old, adv = np.full(N, -12.0, np.float32), np.full(N, 0.5, np.float32)
    want = tune.policy_loss(s, ints(tokens[-last:]), gpu(old[:last]), gpu(adv[:last]), weights=gpu(np.ones(last)),
                            out=torch.empty_like(s))
    pair = tune.preference_loss(s, ints(tokens[-last:]), ints([0, 1, last]), gpu([-12.0, -24.0]), out=torch.empty_like(s))
    for call in ("policy", "preference"):
        scores = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
        scores[-last:] = s
        if call == "policy":
            got = tune.policy_loss(scores, ints(tokens), gpu(old), gpu(adv), weights=gpu(np.ones(N)), out=scores)
            assert bool((got[1][:-last] == 0).all())
            # the rows alone are cut into slices, whose sums are joined
            a, b = host(want[0]), host(got[0][-last:])
            assert (np.abs(a - b) <= 2.0**-18 * np.abs(a)).all()
            a, b = host(want[1]), host(got[1][-last:])
        else:
            got = tune.preference_loss(scores, ints(tokens), ints([N - last, N - last + 1, N]), gpu([-12.0, -24.0]), out=scores)
            assert bool((got[1][:-last] == 0).all())
            a, b = host(pair[1]), host(got[1][-last:])
        assert (np.abs(a - b) <= 2.0**-7 * np.abs(a) + 2.0**-40).all() and np.abs(a).max() > 1e-3
        del scores, got


def test_policy_gradient_against_differences():
    rng = np.random.default_rng(4)
    N, V = 6, 12
    s = rng.normal(0, 1, (N, V))
    tokens, adv = rng.integers(0, V, N), rng.normal(0, 1, N).astype(np.float32)
    heat, w = rng.uniform(0.5, 1.5, N).astype(np.float32), rng.uniform(0.5, 1.5, N).astype(np.float32)
    s = s.astype(np.float32)
    lp = log_softmax(s.astype(float), heat)[0][np.arange(N), tokens]
    old, ref = (lp + 0.05).astype(np.float32), (lp - 0.3).astype(np.float32)
    args = (old.astype(float), adv.astype(float), ref.astype(float), 0.5, 0.2, 0.2, w.astype(float))
    loss = lambda v: policy_want(log_softmax(v, heat)[0], tokens, *args)[0].sum()  # noqa: E731
    _, grad, _ = tune.policy_loss(gpu(s), ints(tokens), gpu(old), gpu(adv), reference=gpu(ref), kl=0.5, weights=gpu(w),
                                  temperature=gpu(heat))
    h = 2.0**-14  # the third derivative times h^2 is below 1e-7
    for n in range(N):
        for v in range(V):
            up, down = s.astype(float), s.astype(float)
            up[n, v] += h
            down[n, v] -= h
            assert abs((loss(up) - loss(down)) / (2 * h) - float(grad[n, v])) < 4e-6


def test_preference_gradient_against_differences():
    rng = np.random.default_rng(4)
    N, V = 9, 11
    s = rng.normal(0, 1, (N, V)).astype(np.float32)
    tokens, starts = rng.integers(0, V, N), np.array([0, 2, 5, 6, 8])
    ref = np.array([-5, -8, -3, -4], np.float32)
    loss = lambda v: preference_want(log_softmax(v, None)[0], tokens, starts, ref.astype(float), 0.7, 0.1)[0].sum()  # noqa: E731
    _, grad, _ = tune.preference_loss(gpu(s), ints(tokens), ints(starts), gpu(ref), beta=0.7, smoothing=0.1)
    h = 2.0**-14
    for n in range(N):
        for v in range(V):
            up, down = s.astype(float), s.astype(float)
            up[n, v] += h
            down[n, v] -= h
            assert abs((loss(up) - loss(down)) / (2 * h) - float(grad[n, v])) < 4e-6


def test_preference_starts_outside_the_rows_are_cut():
    N, V = 6, 20
    scores = score_rows(np.random.default_rng(0), N, V, "f32", masked=0.0)
    tokens, ref = ints(np.arange(N)), gpu([0.0, 0.0])
    a = tune.preference_loss(scores, tokens, ints([0, 3, 6]), ref)
    b = tune.preference_loss(scores, tokens, ints([-7, 3, 2**31 - 1]), ref)
    for s, t in zip(a, b):
        assert torch.equal(s, t)


# ---------------------------------------------------------------------------------- AdamW
F = np.float32


def mixed(h):
    h = h.astype(np.uint64)
    for shift, factor in ((16, 0x85EBCA6B), (13, 0xC2B2AE35), (16, None)):
        h = h ^ (h >> np.uint64(shift))
        if factor:
            h = h * np.uint64(factor) & np.uint64(0xFFFFFFFF)
    return h


def chances(places, k, seed):
    key = mixed(mixed(np.array([k])) ^ np.uint64(seed))
    a = mixed(places.astype(np.uint64) ^ key)
    b = a * np.uint64(0x9E3779B9) & np.uint64(0xFFFFFFFF)
    return [F(v) / F(65536) for v in (a & np.uint64(0xFFFF), a >> np.uint64(16), b >> np.uint64(16))]


def step_of(x, fraction, least):
    e = np.frexp(x)[1] - 1
    return np.ldexp(F(1), np.maximum(np.where(x > 0, e, least), least) - fraction).astype(F)


def drawn_to(x, chance, fraction, least):
    q = step_of(np.abs(x), fraction, least)
    return np.copysign(np.floor(np.abs(x) / q + chance) * q, x).astype(F)


def scale_of(x):
    """(blocks,) scales of magnitudes x (blocks, 256)"""
    most = x.max(1)
    e = (most.view(np.uint32) + 0x1FFFFF >> 23).astype(int)
    return np.ldexp(F(1), np.maximum(e, 37) - 135).astype(F)


class Model:
    """AdamW in float32 as include/ytm.h writes it, on flat arrays."""

    def __init__(self, p, kind, bits):
        self.p, self.kind, self.bits, self.k = p.astype(F), kind, bits, 0
        self.m, self.v = np.zeros_like(self.p), np.zeros_like(self.p)

    def step(self, g, place, seed, lr, b1, b2, eps, decay):
        self.k += 1
        g, m, v = g.astype(F), self.m, self.v
        m = F(b1) * m + F(1 - b1) * g
        v = F(b2) * v + F(1 - b2) * (g * g)
        root = np.sqrt(v)
        rate, cool = F(lr / (1 - b1**self.k)), F(1 / np.sqrt(1 - b2**self.k))
        p = self.p * F(1 - lr * decay) - rate * m / (root * cool + F(eps))
        one, two, three = chances(place + np.arange(p.size), self.k, seed)
        self.exact = p
        if self.kind != "f32":
            p = drawn_to(p, three, *((10, -14) if self.kind == "f16" else (7, -126)))
        self.p = p
        if self.bits == 8:
            pad = -p.size % 256
            block = lambda x: np.concatenate((x, np.zeros(pad, F))).reshape(-1, 256)  # noqa: E731
            s = scale_of(block(np.abs(m)))
            s1 = s.repeat(256)[:p.size]
            m = drawn_to(m / s1, one, 3, -6) * s1
            r = scale_of(block(root))
            s2 = r.repeat(256)[:p.size]
            x = root / s2
            q = step_of(x, 3, -6)
            low = np.floor(x / q) * q
            high = low + q
            up = (x * x - low * low > two * (high * high - low * low)) | ((low == 0) & (x > 0))
            v = np.where(up, high, low) * s2
            self.root, self.scales = v, (s, r)
            v = v * v
        self.m, self.v = m, v


@pytest.mark.parametrize("kind,slope", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(kind, slope, bits):
    """Several steps of tensors of all kinds of sizes."""
    rng = np.random.default_rng(bits)
    sizes = [1, 3, 255, 256, 257, 1000, 4096, 4097, 9001, 5]
    shapes = [(n,) for n in sizes] + [(7, 33), (2, 3, 50), (0,)]
    p = [gpu(rng.normal(0, 0.1, s), kind) for s in shapes]
    g = [gpu(np.zeros(s), slope) for s in shapes]
    models = [Model(host(t).reshape(-1), kind, bits) for t in p]
    a = tune.AdamW(p, g, bits=bits, seed=5)
    for k in range(4):
        for t in g:
            wide = rng.normal(0, 1, t.shape) * np.exp(rng.normal(0, 3, t.shape)) * 1e-3
            t.copy_(gpu(wide * (rng.random(t.shape) < 0.9), slope))
        a.step(lr=0.01, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
        place = 0
        for i, m in enumerate(models):
            m.step(host(g[i]).reshape(-1), place, 5, 0.01, 0.9, 0.99, 1e-6, 0.1)
            place += -(-m.p.size // 256) * 256
            # factors from double roundings: a unit in the last place each, and the sum's
            bound = 2.0**-23 * (3 * np.abs(m.exact) + 0.2)
            off = np.abs(host(p[i]).reshape(-1) - m.p)
            if kind == "f32":
                assert (off <= bound).all(), (k, i)
            else:  # the same draw, but where that rounding passes it
                assert (off > 0).sum() <= 1 + 0.01 * off.size and (off <= 2.01 * ROUND[kind][0] * np.abs(m.p) + 2.0**-24).all(), (k, i)
                m.p = host(p[i]).reshape(-1).astype(F)
            first, second = host(a.first[i]).reshape(-1), host(a.second[i]).reshape(-1)
            if bits == 8:
                np.testing.assert_array_equal(host(a.first_scales[i]), m.scales[0])
                np.testing.assert_array_equal(host(a.second_scales[i]), m.scales[1])
                first = first * m.scales[0].repeat(256)[:first.size]
                second = (second * m.scales[1].repeat(256)[:second.size])
                np.testing.assert_array_equal(second, m.root)
            else:
                np.testing.assert_array_equal(second, m.v)
            np.testing.assert_array_equal(first, m.m)
    assert a.steps.tolist() == [4] * len(p)


def test_adamw_against_64_bits():
    rng = np.random.default_rng(0)
    p0, lr, b1, b2, eps, decay = rng.normal(0, 1, 700).astype(F), 0.02, 0.9, 0.999, 1e-8, 0.05
    p, g = gpu(p0), gpu(np.zeros(700))
    a = tune.AdamW([p], [g])
    x, m, v = p0.astype(float), 0.0, 0.0
    for k in range(1, 11):
        s = rng.normal(0, 1, 700).astype(F)
        g.copy_(gpu(s))
        a.step(lr, (b1, b2), eps, decay)
        m, v = b1 * m + (1 - b1) * s.astype(float), b2 * v + (1 - b2) * s.astype(float)**2
        x = x * (1 - lr * decay) - lr * (m / (1 - b1**k)) / (np.sqrt(v / (1 - b2**k)) + eps)
    # a step rounds p three times and the update, at most lr 10 here, some eight times
    assert (np.abs(host(p) - x) <= 10 * 2.0**-24 * (3 * (np.abs(x) + 0.5) + 8 * 10 * lr)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_past_31_bits(bits):
    """The last elements of a tensor whose elements 31 bits do not count."""
    n, last = 2**31 + 999, 999
    rng = np.random.default_rng(bits)
    start = n - last - (n - last) % 256  # a block's first element
    size = n - start
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    v, s = gpu(rng.normal(0, 0.1, size), "bf16"), gpu(rng.normal(0, 0.1, size), "bf16")
    p[start:], g[start:] = v, s
    a, m = tune.AdamW([p], [g], bits=bits, seed=9), Model(host(v), "bf16", bits)
    for _ in range(2):
        a.step(lr=0.01, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
        m.step(host(s), start, 9, 0.01, 0.9, 0.99, 1e-6, 0.1)
    off = np.abs(host(p[start:]) - m.p)
    assert (off > 0).sum() <= 1 + 0.01 * off.size and (off <= 2.01 * ROUND["bf16"][0] * np.abs(m.p) + 2.0**-24).all()
    first = host(a.first[0][start:])
    if bits == 8:
        first = first * host(a.first_scales[0][start // 256:]).repeat(256)[:size]
    np.testing.assert_array_equal(first, m.m)
    assert not bool(p[:start].any())


def test_adamw_8_bits_keep_means():
    """Averages that move by less than half the distance of two codes a step move all the same: over n elements of one
    value the mean of the stored ones is within six deviations (at most the distance of two codes / 2 sqrt n)."""
    n = 256 * 400
    p, g = gpu(np.zeros(n)), gpu(np.full(n, 1.0))
    a = tune.AdamW([p], [g], bits=8, seed=1)
    a.step(0.0)
    g.fill_(2.0)
    m, v = 0.1, 0.001
    for k in range(30):
        a.step(0.0)
        m, v = 0.9 * m + 0.2, 0.999 * v + 0.004
        first = host(a.first[0]) * host(a.first_scales[0]).repeat(256)
        second = (host(a.second[0]) * host(a.second_scales[0]).repeat(256))**2
        # a step's draws add up: fewer than 31 of them, codes an eighth apart, squares a little more than a quarter
        assert abs(first.mean() - m) <= 6 * np.sqrt(31) * m / 8 / 2 / np.sqrt(n)
        assert abs(second.mean() - v) <= 6 * np.sqrt(31) * v * 0.27 / 2 / np.sqrt(n)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_goes_on_from_its_states(bits):
    rng = np.random.default_rng(1)
    shapes = [(300,), (5, 70)]
    p = [gpu(rng.normal(0, 1, s)) for s in shapes]
    g = [gpu(rng.normal(0, 1, s)) for s in shapes]
    a = tune.AdamW(p, g, bits=bits)
    a.step(0.1)
    q = [t.clone() for t in p]
    b = tune.AdamW(q, g, bits=bits, states={n: [t.clone() for t in s] for n, s in a.states().items()}, steps=a.steps)
    a.step(0.1)
    b.step(0.1)
    for s, t in zip(p + a.first + a.second, q + b.first + b.second):
        assert torch.equal(s.float(), t.float())
    assert b.steps.tolist() == [2, 2]


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_leaves_inactive_tensors(bits):
    rng = np.random.default_rng(1)
    p = [gpu(rng.normal(0, 1, 500)) for _ in range(5)]
    g = [gpu(rng.normal(0, 1, 500)) for _ in range(5)]
    a, was = tune.AdamW(p, g, bits=bits), [t.clone() for t in p]
    a.step(torch.tensor(0.1, device="cuda"), active=torch.tensor([True, False, True, False, False], device="cuda"))
    assert a.steps.tolist() == [1, 0, 1, 0, 0]
    for i, (s, t) in enumerate(zip(p, was)):
        assert torch.equal(s, t) == (i not in (0, 2))
        assert bool((a.first[i].float() == 0).all()) == (i not in (0, 2))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_values_that_are_not_finite_stay_in_their_element(bits):
    n = 600
    rng = np.random.default_rng(1)
    v = rng.normal(0, 1, n).astype(F)
    p, q, g, h = gpu(np.ones(n)), gpu(np.ones(n)), gpu(v), gpu(v)
    a, b = tune.AdamW([p], [g], bits=bits), tune.AdamW([q], [h], bits=bits)
    bad = [3, 300, 301]
    g[3], g[300], g[301] = float("nan"), float("inf"), -float("inf")
    h[bad] = 0.0
    for _ in range(2):
        a.step(0.1)
        b.step(0.1)
    good = np.setdiff1d(np.arange(n), bad)
    assert torch.equal(p[good], q[good]) and torch.equal(a.second[0].float()[good], b.second[0].float()[good])
    assert not bool(torch.isfinite(p[bad]).any())


# ----------------------------------------------------------------- together, streams, graphs
def test_learning_together():
    """Adapters that learn to give the preferred answers: adapt, loss, gradient and step as they are used."""
    C, K, N, users = 200, 50, 40, 3
    rng = np.random.default_rng(0)
    bits = decode.pack_outputs(rng.random((N, C)) < 0.3)
    codes, scales = decode.pack_weights(rng.integers(-5, 6, (C, K)).astype(F))
    base = decode.readout(bits, codes, scales, clauses=C)
    which = ints(np.where(np.arange(N) % 4 == 3, -1, np.arange(N) % 4))
    tokens, heat = ints(rng.integers(0, K, N)), gpu(np.full(N, 10.0))
    adapters = tune.Adapters(users + 2, C, K, rank=8, bits=8)
    before = [t.clone() for t in (adapters.down, adapters.up)]
    for step in range(3):
        scores = base.clone()
        hidden = adapters.adapt(scores, bits, which)
        want = host(base)
        for n in range(N):
            a = int(which[n])
            if a >= 0:
                want[n] += host(adapters.up[a]) @ host(hidden[n])
        assert np.abs(host(scores) - want).max() <= 2.0**-20 * np.abs(want).max()
        old = gpu(np.full(N, -4.0))
        _, grad, lp = tune.policy_loss(scores, tokens, old, gpu(np.ones(N)), temperature=heat, out=scores)
        adapters.learn(grad, bits, which, hidden, lr=1e-2)
        for a in range(users, users + 2):  # nobody's adapters
            assert torch.equal(adapters.down[a], before[0][a]) and torch.equal(adapters.up[a], before[1][a])
    assert not torch.equal(adapters.up[:users], before[1][:users])
    assert not torch.equal(adapters.down[:users], before[0][:users])
    assert adapters.optimizer.steps.tolist() == [3] * 6 + [0] * 4


def everything(c, scores, tokens, old, adv, starts, ref, grad_to, opt, lr):
    """One pass of all operators; what they give."""
    hidden = torch.empty(c.N, c.r, device="cuda")
    out = tune.adapt(scores, c.x, c.down, c.up, c.which, c.scale, hidden=hidden)
    a = tune.policy_loss(out, tokens, old, adv)
    b = tune.preference_loss(out, tokens, starts, ref)
    d = tune.adapt_gradient(a[1], c.x, c.down, c.up, c.which, hidden, c.scale, out=grad_to)
    opt.step(lr)
    return [out, hidden, *a, *b, *d, *opt.first, *opt.second]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("N,V", [(40, 300), (300, 4100), (3, 40000)])
def test_graph_replays(N, V, bits):
    """Captured once, replayed with other inputs and eager work between the replays."""
    rng = np.random.default_rng(N)

    def inputs():
        s = rng.integers(-4, 5, (N, V)).astype(F)
        return gpu(s), ints(rng.integers(0, V, N)), gpu(np.full(N, -4.0)), gpu(rng.normal(0, 1, N))

    def setup():
        c = Case(N, 100, V, 6, 4, exact=False)
        grads = torch.zeros_like(c.down), torch.zeros_like(c.up)
        return c, grads, tune.AdamW([c.down, c.up], list(grads), bits=bits, seed=3)

    starts, ref = ints([0, N // 3, N]), gpu([-30.0, -40.0])
    (c, grads, opt), (e, e_grads, e_opt) = setup(), setup()
    held, lr = inputs(), torch.tensor(0.01, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        everything(c, *held, starts, ref, grads, opt, lr)
    torch.cuda.current_stream().wait_stream(stream)
    everything(e, *held, starts, ref, e_grads, e_opt, lr)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = everything(c, *held, starts, ref, grads, opt, lr)
    for k in range(3):
        new = inputs()
        for s, t in zip(held, new):
            s.copy_(t)
        lr.fill_(0.01 * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = everything(e, *new, starts, ref, e_grads, e_opt, lr)
        torch.cuda.synchronize()
        for s, t in zip(captured + [c.down, c.up, opt.steps], eager + [e.down, e.up, e_opt.steps]):
            assert torch.equal(s.float(), t.float()), k


@pytest.mark.parametrize("bits", [32, 8])
def test_learning_in_a_graph(bits):
    """A whole step of Adapters captured: corrected scores, loss, gradient, optimiser, with users that change."""
    C, K, N, users = 100, 40, 30, 4
    rng = np.random.default_rng(0)
    bits_in = decode.pack_outputs(rng.random((N, C)) < 0.3)
    base, adv = gpu(rng.normal(0, 3, (N, K))), gpu(rng.normal(0, 1, N))
    tokens, which, old = ints(rng.integers(0, K, N)), ints(rng.integers(0, users - 1, N)), gpu(np.full(N, -3.0))
    models = [tune.Adapters(users, C, K, rank=5, bits=bits, seed=4) for _ in range(2)]

    def step(m):
        scores = base.clone()
        hidden = m.adapt(scores, bits_in, which)
        _, grad, lp = tune.policy_loss(scores, tokens, old, adv, out=scores)
        m.learn(grad, bits_in, which, hidden, lr=0.05)
        return lp

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(models[0])
    torch.cuda.current_stream().wait_stream(stream)
    step(models[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(models[0])
    for k in range(3):
        which.copy_(ints(rng.integers(-1, users - k, N)))
        graph.replay()
        torch.cuda.synchronize()
        eager = step(models[1])
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)
        for a, b in zip((models[0].down, models[0].up, models[0].optimizer.steps),
                        (models[1].down, models[1].up, models[1].optimizer.steps)):
            assert torch.equal(a, b), k


def test_two_streams_at_once():
    """Calls of two streams, with workspaces of their own."""
    cases = [Case(300, 500, 900, 16, 5, seed=q) for q in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for q, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                out, hidden = c.adapt()
                got[q].append((out, hidden, tune.preference_loss(out, c.which, ints([0, 150, 300]), gpu([0.0, 0.0]))))
    torch.cuda.synchronize()
    for q, c in enumerate(cases):
        for out, hidden, loss in got[q]:
            np.testing.assert_array_equal(host(out), c.out)
            np.testing.assert_array_equal(host(hidden), c.hidden)
            assert torch.equal(loss[1], got[q][0][2][1])


@pytest.mark.parametrize("call", ["adapt", "gradient", "policy", "preference"])
def test_what_is_written_must_not_overlap_what_is_read(call):
    c = Case(20, 64, 64, 4, 2, "f32")
    hidden = torch.empty(20, 4, device="cuda")
    flat = torch.zeros(20 * 64 + 8, device="cuda")
    near, off = flat[:20 * 64].view(20, 64), flat[8:].view(20, 64)
    near.copy_(c.scores)
    tokens, rows = ints(np.zeros(20)), gpu(np.zeros(20))
    with pytest.raises(ValueError, match="overlap"):
        if call == "adapt":
            tune.adapt(near, c.x, c.down, c.up, c.which, out=off)
        elif call == "gradient":
            tune.adapt_gradient(near, c.x, c.down, c.up, c.which, hidden,
                                out=(off.reshape(-1)[:512].view(2, 4, 64), torch.empty_like(c.up)))
        elif call == "policy":
            tune.policy_loss(near, tokens, rows, rows, out=off)
        else:
            tune.preference_loss(near, tokens, ints([0, 10, 20]), gpu([0.0, 0.0]), out=off)


def test_adamw_refuses_what_overlaps():
    flat = torch.zeros(1000, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        tune.AdamW([flat[:600], flat[500:]], [torch.zeros(600, device="cuda"), torch.zeros(500, device="cuda")])
    with pytest.raises(ValueError, match="overlap"):
        tune.AdamW([flat[:600]], [flat[300:900]])
    shared = torch.zeros(500, device="cuda")
    tune.AdamW([flat[:500], flat[500:]], [shared, shared]).step()
