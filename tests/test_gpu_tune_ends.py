"""The adapting and learning operators at the ends of their ranges: memory that is not an operand's own, numbers at
the ends of their types, what is left out, and objects that are copied."""
import copy
import io
import pickle

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ytm_amd = pytest.importorskip("ytm_amd")
from ytm_amd import tune  # noqa: E402

from test_gpu_tune import TYPES, Case, gpu, host, ints, spread, untouched, within  # noqa: E402


# ------------------------------------------------------------------------------- adapters
@pytest.mark.parametrize("w", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,K,r", [(20, 128, 48), (300, 64, 48), (17, 192, 80), (5, 64, 112), (40, 130, 144), (9, 64, 240),
                                   (20, 128, 64), (20, 128, 32)])
def test_adapt_reads_no_weights_behind_a_row(N, K, r, w):
    """Ranks of whole 16s: NaN between the rows of up and in the adapters between those that rows name."""
    c = Case(N, 100, K, r, 3, "bits", w, which=np.arange(N) % 4 - 1)
    memory = torch.full((5, K, r + 19), float("nan"), dtype=TYPES[w], device="cuda")
    up = memory[::2, :, :r]
    up.copy_(c.up)
    memory[::2, :, r:] = float("nan")
    hidden = torch.empty(N, r, device="cuda")
    out = tune.adapt(c.scores, c.x, c.down, up, c.which, c.scale, hidden=hidden)
    np.testing.assert_array_equal(host(hidden), c.hidden)
    np.testing.assert_array_equal(host(out), c.out)
    # rows one after the other: what follows one is the next output's, which is not finite
    c.up[:, 1::2] = float("inf")
    c.up[1] = float("nan")
    out = host(tune.adapt(c.scores, c.x, c.down, c.up, c.which, c.scale))
    clean = c.numbers != 1
    np.testing.assert_array_equal(out[clean][:, 0::2], c.out[clean][:, 0::2])


def among_nan(t, pad, offset):
    """The same tensor with NaN between its rows and around it."""
    *front, width = t.shape
    rows = int(np.prod(front))
    memory = torch.full((rows * (width + pad) + offset + 8,), float("nan"), dtype=t.dtype, device="cuda")
    out = memory[offset:offset + rows * (width + pad)].view(*front, width + pad)[..., :width]
    out.copy_(t)
    return out


@pytest.mark.parametrize("x,w,kind", [("bits", "f32", "f32"), ("f32", "f32", "bf16"), ("f16", "f16", "f16"),
                                      ("bf16", "bf16", "bf16"), ("f32", "bf16", "f32")])
@pytest.mark.parametrize("N,C,K,r,M,pad,offset", [(1, 7, 3, 1, 1, 1, 1), (33, 130, 64, 16, 3, 5, 3), (20, 259, 129, 48, 2, 3, 0),
                                                  (300, 65, 192, 33, 9, 1, 7), (700, 128, 70, 112, 40, 8, 8),
                                                  (260, 200, 100, 24, 1, 2, 5)])
def test_what_lies_between_rows_is_not_used(N, C, K, r, M, pad, offset, x, w, kind):
    c = Case(N, C, K, r, M, x, w)
    rng = np.random.default_rng(3)
    grad, h = rng.integers(-1, 2, (N, K)).astype(float), rng.integers(-2, 3, (N, r)).astype(float)
    clauses = c.x if x == "bits" else among_nan(c.x, pad, offset)
    down, up, scores = (among_nan(t, pad, offset) for t in (c.down, c.up, c.scores))
    hidden = torch.empty(N, r, device="cuda")
    out = tune.adapt(scores, clauses, down, up, c.which, c.scale, hidden=hidden)
    np.testing.assert_array_equal(host(hidden), c.hidden)
    np.testing.assert_array_equal(host(out), c.out)
    wants, _ = c.gradients(grad, h)
    got = tune.adapt_gradient(among_nan(gpu(grad, kind), pad, offset), clauses, down, up, c.which,
                              among_nan(gpu(h), pad, offset), c.scale)
    for t, want in zip(got, wants):
        np.testing.assert_array_equal(host(t), host(torch.from_numpy(want).float().to(TYPES[w])))


@pytest.fixture
def other_defaults():
    torch.set_default_device("cuda")
    torch.set_default_dtype(torch.bfloat16)
    yield
    torch.set_default_device(None)
    torch.set_default_dtype(torch.float32)


@pytest.mark.parametrize("bits", [32, 8])
def test_torchs_defaults_change_nothing(bits, request):
    def learnt():
        rng = np.random.default_rng(0)
        a = tune.Adapters(3, 50, 20, rank=4, bits=bits, seed=2)
        scores, which = gpu(rng.normal(0, 1, (30, 20))), ints(np.arange(30) % 3 - 1)
        x = gpu(rng.normal(0, 1, (30, 50)))
        hidden = a.adapt(scores, x, which)
        _, grad, lp = tune.policy_loss(scores, ints(np.arange(30) % 20), gpu(np.zeros(30)), gpu(np.ones(30)))
        a.learn(grad, x, which, hidden)
        return [a.down, a.up, hidden, grad, lp]

    want = learnt()
    request.getfixturevalue("other_defaults")
    for s, t in zip(want, learnt()):
        assert s.dtype == t.dtype and torch.equal(s, t)


@pytest.mark.parametrize("w,kind", [("f16", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("N,C,K,r,M", [(1, 500, 40, 4, 1), (40, 777, 129, 16, 9), (300, 333, 65, 40, 4), (700, 130, 90, 8, 300)])
def test_float32_gradients_of_16_bit_adapters(N, C, K, r, M, w, kind):
    """Sums that 16 bits hold nothing, or a bit or two, of."""
    c = Case(N, C, K, r, M, "bits", w, exact=False)
    rng = np.random.default_rng(2)
    grad = gpu(rng.normal(0, 1e-8, (N, K)), kind if kind == "bf16" else "f32")
    hidden = gpu(rng.normal(0, 1, (N, r)))
    want, size = c.gradients(host(grad), host(hidden))
    to = tuple(spread(torch.zeros(*t.shape, device="cuda"), 3, 1) for t in (c.down, c.up))
    got = tune.adapt_gradient(grad, c.x, c.down, c.up, c.which, hidden, c.scale, out=to)
    assert got[0] is to[0] and got[1] is to[1] and untouched(to[0], 3, 1) and untouched(to[1], 3, 1)
    within(got[0], want[0], size[0], N + K + 1, "f32")
    within(got[1], want[1], size[1], N + 1, "f32")
    narrow = tune.adapt_gradient(grad, c.x, c.down, c.up, c.which, hidden, c.scale)
    for s, t in zip(got, narrow):
        assert t.dtype is TYPES[w] and torch.equal(s.to(t.dtype), t)


def test_float16_adapters_learn_from_unlikely_answers():
    """A mean over a batch and many outputs, some of whose sums float16 makes 0.  An answer's probability is
    exp(3 z) / (5000 exp(9 / 2)), z normal, so the sums of 64 rows' are a few 10^-6 in the median, and a few in a
    thousand of the 20000 are below 2^-25."""
    N, C, K, r = 64, 100, 5000, 4
    rng = np.random.default_rng(0)
    a = tune.Adapters(1, C, K, rank=r, dtype=torch.float16)
    scores, x = gpu(rng.normal(0, 3, (N, K))), gpu(rng.normal(0, 1, (N, C)), "f16")
    which = ints(np.zeros(N))
    hidden = a.adapt(scores, x, which)
    tokens = ints(rng.integers(0, 10, N))
    _, grad, lp = tune.policy_loss(scores, tokens, gpu(np.zeros(N)), gpu(np.ones(N)))
    _, grad, _ = tune.policy_loss(scores, tokens, lp, gpu(np.ones(N)))
    a.learn(grad, x, which, hidden, lr=0.01, eps=1e-15, weight_decay=0.0)
    sums = a.gradients[1][0]
    assert sums.dtype is torch.float32 and bool((sums.abs() < 2.0**-25).any())
    # the first step is as long for all, against the gradient
    assert bool((a.up[0].float() * sums < 0).all()) and float((a.up[0].float().abs() - 0.01).abs().max()) < 2e-5


# --------------------------------------------------------------------------------- losses
def both_losses(scores, tokens, **kw):
    """(losses, gradient, log probabilities) of the policy's loss, gradient and log probabilities of a preference's."""
    N = scores.shape[0]
    policy = tune.policy_loss(scores, ints(tokens), gpu(np.zeros(N)), gpu(np.ones(N)), weights=gpu(np.ones(N)), **kw)
    starts, reference = ints([0, *[1] * (N > 1), N, *[N] * (N < 2)]), gpu([0.0, 0.0])
    return policy + tune.preference_loss(scores, ints(tokens), starts, reference, **kw)[1:]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,V", [(2, 40), (2, 5000), (300, 4100), (2, 70000)])
def test_an_infinite_temperature_leaves_masks_in_place(N, V, kind):
    """All answers that are not masked are alike; a probability is 1 / V to the rounding of a sum of V ones."""
    s = np.random.default_rng(0).normal(0, 3, (N, V))
    s[:, ::3] = -np.inf
    s[1, :3] = np.nan, 2.0, 6e4
    scores, tokens = gpu(s, kind), np.full(N, 2)
    heat = np.full(N, np.inf)
    losses, grad, lp, pair_grad, said = both_losses(scores, tokens, temperature=gpu(heat))
    count = np.isfinite(s).sum(1)
    # 16 units: of a sum of ones in chains of at most V / 64 + 64 that are exact below 2^24, of its logarithm, two
    # powers and three products
    assert (np.abs(host(lp) + np.log(count)) <= 2.0**-20 * np.log(count)).all()
    assert bool(torch.isfinite(grad).all()) and bool(torch.isfinite(pair_grad).all()) and bool(torch.isfinite(said).all())
    assert not bool(grad[:, ::3].any()) and not bool(pair_grad[:, ::3].any())
    assert float(grad[0].abs().max()) < 1e-38  # nothing that is divided by an infinite temperature is left


@pytest.mark.parametrize("N,V", [(8, 40), (8, 5000), (8, 70000)])
def test_rows_of_weight_0_are_left_out(N, V):
    """Rows that fill a batch, with numbers whose ratio or distance is infinite or NaN."""
    rng = np.random.default_rng(0)
    scores, tokens = gpu(rng.normal(0, 3, (N, V))), rng.integers(0, V, N)
    old, adv, reference, weights = np.full(N, -4.0), np.ones(N), np.full(N, -5.0), np.full(N, 0.25)
    old[1], old[2], adv[3], reference[4], reference[5] = -1e4, np.nan, np.nan, 1e4, np.inf
    old[6], adv[6] = -np.inf, -1.0
    weights[1:7] = 0.0
    weights[6] = -0.0
    losses, grad, lp = tune.policy_loss(scores, ints(tokens), gpu(old), gpu(adv), reference=gpu(reference), kl=0.1,
                                        weights=gpu(weights))
    assert not bool(losses[1:7].any()) and not bool(grad[1:7].any())
    assert bool((lp < 0).all()) and bool(torch.isfinite(grad).all())
    # the others, as if they were alone
    ends = [0, 7]
    want = tune.policy_loss(scores[::7], ints(tokens[ends]), gpu(old[ends]), gpu(adv[ends]),
                            reference=gpu(reference[ends]), kl=0.1, weights=gpu(weights[ends]))
    for s, t in zip((losses, grad, lp), want):
        # rows longer than a slice are cut otherwise, and joined: sums of exponentials to 2^-20, the log's to 2^-22
        assert float((s[::7] - t).abs().max()) <= 2.0**-18 * (1 if V >= 32768 else 0)
        assert float(t.abs().max()) > 1e-5


@pytest.mark.parametrize("V", [40, 5000, 70000])
def test_numbers_that_are_nan_are_not_hidden(V):
    """And stay in their rows; a ratio past float32 of an advantage of 0 is none."""
    N = 6
    rng = np.random.default_rng(0)
    scores, tokens = gpu(rng.normal(0, 3, (N, V))), rng.integers(0, V, N)
    old, adv, reference = np.full(N, -4.0), np.ones(N), np.full(N, -5.0)
    old[1], adv[2], reference[3] = np.nan, np.nan, np.nan
    old[4], adv[4] = -1e4, 0.0
    for kl in (0.0, 0.1):
        losses, grad, lp = tune.policy_loss(scores, ints(tokens), gpu(old), gpu(adv), reference=gpu(reference), kl=kl)
        bad = [1, 2] + [3] * (kl > 0)
        good = [n for n in range(N) if n not in bad]
        assert bool(torch.isnan(losses[bad]).all()) and bool(torch.isnan(grad[bad]).all())
        assert bool(torch.isfinite(losses[good]).all()) and bool(torch.isfinite(grad[good]).all())
        assert bool(torch.isfinite(lp).all())
        if not kl:
            assert float(losses[4]) == 0.0 and not bool(grad[4].any())


@pytest.mark.parametrize("pairs,V", [(3, 40), (200, 300), (3, 40000)])
def test_references_that_a_mask_made_infinite(pairs, V):
    """A sequence that the reference cannot say: preferred, its pair is won and its loss 0; the other way it is lost."""
    N = 2 * pairs
    scores, tokens = gpu(np.random.default_rng(0).normal(0, 3, (N, V))), ints(np.arange(N) % V)
    reference = np.full(N, -5.0)
    reference[0] = reference[3] = -np.inf
    starts = ints(np.arange(N + 1))
    for smoothing, won, lost in ((0.0, 0.0, np.inf), (1.0, np.inf, 0.0), (0.5, np.inf, np.inf)):
        losses, grad, _ = tune.preference_loss(scores, tokens, starts, gpu(reference), smoothing=smoothing)
        assert float(losses[0]) == won and float(losses[1]) == lost
        assert bool(torch.isfinite(losses[2:]).all()) and bool(torch.isfinite(grad).all())
        # a loss that is as small as it gets has no slope
        assert not bool(grad[:2].any()) if won == 0.0 else bool(grad[:2].any())
        assert not bool(grad[2:4].any()) if lost == 0.0 else bool(grad[2:4].any())


# ---------------------------------------------------------------------------------- AdamW
@pytest.mark.parametrize("size", [1e-10, 1e-14, 1e-17, 1e-18])
def test_second_states_above_zero_stay_above_it(size):
    """8 bits, eps 0: gradients whose squares float32 holds, of very different sizes in a block, and none after."""
    rng = np.random.default_rng(0)
    n = 256 * 6 + 100
    g = gpu(size * 10.0 ** rng.uniform(-1, 0, n) * rng.choice([-1, 1], n))
    g[::256] *= 1.0 / 16  # codes that are next to 0
    p = gpu(np.ones(n))
    a = tune.AdamW([p], [g], bits=8, seed=3)
    root = lambda: host(a.second[0]) * host(a.second_scales[0]).repeat(256)[:n]  # noqa: E731
    for k in range(4):
        a.step(0.01, eps=0.0)
        assert bool(torch.isfinite(p).all()) and (root() > 0).all(), k
        assert (np.float32(root()) ** 2 >= 2.0**-126).all() and float(a.second_scales[0].min()) >= 2.0**-54, k
        assert float((p - 1).abs().max()) <= 4 * 0.011 * (k + 1), k
        if k == 0:
            g.zero_()


def test_blocks_of_zeros_keep_their_scale():
    p, g = gpu(np.ones(600)), gpu(np.zeros(600))
    g[300] = 1.0
    a = tune.AdamW([p], [g], bits=8)
    a.step(0.01)
    assert a.second_scales[0].tolist()[::2] == a.first_scales[0].tolist()[::2] == [2.0**-98] * 2
    assert float(a.second_scales[0][1]) > 2.0**-54 and not bool(a.second[0][:256].float().any())


def test_float32_steps_are_rounded_as_they_are_written():
    """The first step of parameters that are 0, in numpy's float32."""
    F, n = np.float32, 100003
    rng = np.random.default_rng(0)
    g = (rng.normal(0, 1, n) * np.exp(rng.normal(0, 5, n))).astype(F)
    p, slopes = gpu(np.zeros(n)), gpu(g)
    a = tune.AdamW([p], [slopes])
    a.step(lr=0.01, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
    m, v = F(1 - 0.9) * g, F(1 - 0.99) * (g * g)
    by = np.sqrt(v) * F(1 / np.sqrt(1 - 0.99)) + F(1e-6)
    want = F(0) * F(1 - 0.01 * 0.1) - F(0.01 / (1 - 0.9)) * m / by
    np.testing.assert_array_equal(p.cpu().numpy(), want)


# --------------------------------------------------------------------------------- copies
def saved(a):
    f = io.BytesIO()
    torch.save(a, f)
    f.seek(0)
    return torch.load(f, weights_only=False)  # what this test wrote itself


def learn(a, seed):
    rng = np.random.default_rng(seed)
    x, which, grad = gpu(rng.normal(0, 1, (30, 50))), ints(rng.integers(-1, 3, 30)), gpu(rng.normal(0, 1, (30, 20)))
    hidden = a.adapt(gpu(np.zeros((30, 20))), x, which)
    a.learn(grad, x, which, hidden, lr=0.05)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("copied", [copy.deepcopy, lambda a: pickle.loads(pickle.dumps(a)), saved])
def test_copies_of_adapters_learn_apart(copied, bits):
    a = tune.Adapters(3, 50, 20, rank=4, bits=bits, seed=2, scale=0.5)
    learn(a, 1)
    frozen = [t.clone() for t in (a.down, a.up, *a.optimizer.first)]
    b = copied(a)
    learn(b, 2)
    for s, t in zip(frozen, (a.down, a.up, *a.optimizer.first)):
        assert torch.equal(s.float(), t.float())
    assert not torch.equal(b.up, a.up) and not torch.equal(b.down, a.down)
    learn(a, 2)  # the same step from the same states
    for s, t in zip((a.down, a.up, *a.optimizer.first, *a.optimizer.second, a.optimizer.steps),
                    (b.down, b.up, *b.optimizer.first, *b.optimizer.second, b.optimizer.steps)):
        assert torch.equal(s.float(), t.float())
    del a
    learn(b, 3)


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_of_adamw_step_their_own(bits):
    a = tune.AdamW([gpu(np.ones(500))], [gpu(np.ones(500))], bits=bits, seed=1)
    a.step(0.1)
    was, b = a.parameters[0].clone(), copy.deepcopy(a)
    b.step(0.1)
    assert torch.equal(a.parameters[0], was) and not torch.equal(b.parameters[0], was)
    a.step(0.1)
    assert torch.equal(a.parameters[0], b.parameters[0]) and a.steps.tolist() == b.steps.tolist() == [2]


# ---------------------------------------------------------------------------------- graphs
def test_learning_of_many_rows_in_a_graph():
    """More rows than one block sees, replayed with users that change and eager work between the replays."""
    C, K, N, users = 64, 12, 20000, 40
    rng = np.random.default_rng(0)
    x, grad = gpu(rng.normal(0, 1, (N, C))), gpu(rng.normal(0, 1, (N, K)))
    which = ints(rng.integers(0, 10, N))
    models = [tune.Adapters(users, C, K, rank=3, seed=4) for _ in range(2)]

    def step(m):
        hidden = m.adapt(torch.zeros(N, K, device="cuda"), x, which)
        m.learn(grad, x, which, hidden, lr=0.05)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(models[0])
    torch.cuda.current_stream().wait_stream(stream)
    step(models[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(models[0])
    for k in range(4):
        which.copy_(ints(rng.integers(10 * k - 3, 10 * k + 10, N)))
        graph.replay()
        torch.cuda.synchronize()
        step(models[1])
        torch.cuda.synchronize()
        for s, t in zip((models[0].down, models[0].up, models[0].optimizer.steps),
                        (models[1].down, models[1].up, models[1].optimizer.steps)):
            assert torch.equal(s, t), k
