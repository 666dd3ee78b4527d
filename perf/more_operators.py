"""Cases for timing the operators that adapt a model's answers and learn from them: low-rank
adapters of many requests beside the readout and their gradient, the losses of drawn and of compared
answers with the gradient of the scores, and the AdamW step over many tensors.

Each case is one call as a program that serves or teaches makes it.  With `own` false the operators
are computed in their plain form, elementary torch operations in float32; with `own` true by
ytm_amd.tune.  Models' sizes are those of the benchmark configurations (2000 to 20000 clauses, 10
classes, 10000 words); larger answer sets and batches are generic.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
E4M3 = torch.float8_e4m3fn
BLOCK = 256  # elements of a state in 8 bits that share a scale
SCALE, KL, CLIP, BETA, SMOOTHING = 2.0, 0.05, 0.2, 0.1, 0.05
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one image of one user, the flat image model's 2000 clauses and 10 classes: latency
        dict(name="adapt_digits", op="adapt", n=1, c=2000, k=10, r=8, m=16, x="bits", weights="float32",
             scores="float32"),
        # the next word of 48 users' texts at once, most of them with an adapter of their own
        dict(name="adapt_words", op="adapt", n=48, c=10000, k=10000, r=16, m=64, x="bits", weights="float16",
             scores="float32"),
        # a set of documents of a few tenants, clause outputs averaged over models, the largest clause count
        dict(name="adapt_documents", op="adapt", n=512, c=20000, k=10000, r=32, m=8, x="bfloat16", weights="bfloat16",
             scores="float32"),
        # what a user's 40 marked words teach: latency of a small step
        dict(name="teach_words", op="gradient", n=40, c=10000, k=10000, r=16, m=1, x="bits", weights="float32",
             scores="float32"),
        # a training batch of several tenants, odd sizes, 16-bit weights and gradients
        dict(name="teach_tenants", op="gradient", n=2048, c=9973, k=10007, r=32, m=8, x="bits", weights="bfloat16",
             scores="bfloat16"),
        # one user's drawn words, few rows
        dict(name="policy_words", op="policy", n=24, v=10000, scores="float32", out="float32", temperature=True),
        # a training batch of drawn words over a large vocabulary, in 16 bits
        dict(name="policy_batch", op="policy", n=1024, v=131072, scores="bfloat16", out="bfloat16", temperature=False),
        # two answers of a few words, one preferred
        dict(name="preference_pair", op="preference", n=33, v=10000, pairs=1, scores="float32", out="float32",
             temperature=False),
        # a training batch of compared answers, an odd number of words
        dict(name="preference_batch", op="preference", n=2048, v=32001, pairs=16, scores="bfloat16", out="bfloat16",
             temperature=True),
        # one user's adapter and bias of the flat image model: latency
        dict(name="adamw_user", op="adamw", adapters=1, c=2000, k=10, r=8, parameters="float32", bits=32),
        # the adapters of 64 users at once, states in 8 bits
        dict(name="adamw_users", op="adamw", adapters=64, c=10000, k=10007, r=16, parameters="float32", bits=8),
        # the largest, 16-bit parameters
        dict(name="adamw_tenants", op="adamw", adapters=64, c=20000, k=10000, r=32, parameters="bfloat16", bits=32),
    ]


MOST = 1.2e9  # bytes of the largest listed case, which no drawn one passes


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    types = ["float32", "float16", "bfloat16"]
    op = rng.choice(["adapt", "adapt", "gradient", "gradient", "policy", "preference", "adamw"])
    if op in ("adapt", "gradient"):
        n, c, k = log(1, 512 if op == "adapt" else 2048), log(200, 20000), log(10, 32768)
        r = rng.choice([1, 2, 4, 5, 8, 8, 16, 16, 24, 32, 32, 64])
        m = log(1, 64 if op == "adapt" else 8)
        k = min(k, 40000000 // n, 30000000 // (m * r))
        w = rng.choice(types)
        return dict(op=op, n=n, c=c, k=k, r=r, m=m, x=rng.choice(["bits", "bits", w, "float32"]), weights=w,
                    scores=rng.choice(["float32", w if w != "float16" or op == "adapt" else "float32"]))
    if op == "adamw":
        r, c, k, a = rng.choice([1, 4, 7, 8, 16, 32, 64]), log(200, 20000), log(10, 32768), log(1, 64)
        a = max(1, min(a, 40000000 // (r * (c + k))))
        return dict(op=op, adapters=a, c=c, k=k, r=r, parameters=rng.choice(types), bits=rng.choice([8, 8, 32]))
    n, v, x = log(4, 2048), log(10, 131072), rng.choice(["float32", "bfloat16"])
    n = max(4, min(n, 100000000 // v))
    case = dict(op=op, n=n, v=v, scores=x, out=rng.choice(["float32", x]), temperature=rng.random() < 0.5)
    return dict(case, pairs=log(1, max(1, n // 4))) if op == "preference" else case


# ---------------------------------------------------------------------------------- inputs
def words(n, c, share, g):
    """Clause outputs as int32 words, bit b of word j clause 32 j + b."""
    w = torch.zeros(n, -(-c // 32), dtype=torch.int64, device="cuda")
    for b in range(32):
        w |= (torch.rand(w.shape, generator=g, device="cuda") < share).long() << b
    if c % 32:
        w[:, -1] &= (1 << c % 32) - 1
    return (w - (w >> 31 << 32)).to(torch.int32)


def normal(*shape, g):
    return torch.randn(*shape, generator=g, device="cuda")


def uniform(*shape, g):
    return torch.rand(*shape, generator=g, device="cuda")


def adapters(case, s, g):
    n, c, k, r, m, w = case["n"], case["c"], case["k"], case["r"], case["m"], TYPES[case["weights"]]
    s["down"] = (normal(m, r, c, g=g) / math.sqrt(c)).to(w)
    s["up"] = (normal(m, k, r, g=g) * 0.1).to(w)
    # the r-th busiest tenant has about 1 / r of the rows, one row in 20 has no adapter
    which = (m ** uniform(n, g=g) * (1 + 1e-6)).to(torch.int32).clamp_(1, m) - 1
    s["which"] = torch.where(uniform(n, g=g) < (0.05 if n > 1 else 0.0), -1, which).to(torch.int32)
    if case["x"] == "bits":  # a tenth of the clauses fire
        s["x_in"] = words(n, c, 0.1, g)
    else:  # shares of models or patches in which a clause fires, most of them zero
        x = uniform(n, c, g=g)
        s["x_in"] = torch.where(x < 0.3, uniform(n, c, g=g), 0.0).to(TYPES[case["x"]])


def answered(case, s, g):
    """Scores as a readout gives them, the drawn answer of each row, -1 where a row is none."""
    n, v = case["n"], case["v"]
    x = normal(n, v, g=g).mul_(3.0)
    x += 6.0 * (uniform(n, v, g=g) < 20.0 / v)
    x = s["in"] = x.to(TYPES[case["scores"]])
    s["temperature"] = 0.5 + uniform(n, g=g) if case["temperature"] else None
    z = x.float() if s["temperature"] is None else x.float() / s["temperature"][:, None]
    u = uniform(n, v, g=g).clamp_(1e-7, 1.0 - 1e-7)
    t = (z - torch.log(-torch.log(u))).argmax(1)
    s["lp"] = z.gather(1, t[:, None])[:, 0] - torch.logsumexp(z, 1)
    s["tokens"] = torch.where(uniform(n, g=g) < 0.03, -1, t).to(torch.int32)
    s["to"] = torch.empty(n, v, dtype=TYPES[case["out"]], device="cuda")


def places(case):
    """(element count, offset) of each tensor in one buffer: down, up and bias of each adapter, each at a
    multiple of 256."""
    at, found = 0, []
    for _ in range(case["adapters"]):
        for size in (case["r"] * case["c"], case["k"] * case["r"], case["k"]):
            found.append((size, at))
            at += -(-size // BLOCK) * BLOCK
    return found, at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "adapt":
        adapters(case, s, g)
        s["in"] = (normal(case["n"], case["k"], g=g) * 3.0).to(TYPES[case["scores"]])
        s["to"] = torch.empty(case["n"], case["k"], device="cuda")
    elif case["op"] == "gradient":
        adapters(case, s, g)
        # what a loss leaves: small everywhere, large at one word of each row
        n, k = case["n"], case["k"]
        x = normal(n, k, g=g).mul_(1e-3 / math.sqrt(k))
        x[torch.arange(n, device="cuda"), torch.randint(0, k, (n,), generator=g, device="cuda")] = 1e-3 * normal(n, g=g)
        s["in"] = x.to(TYPES[case["scores"]])
        s["hidden"] = normal(n, case["r"], g=g) * (s["which"] >= 0)[:, None]
        w = TYPES[case["weights"]]
        s["to"] = tuple(torch.empty(s[t].shape, dtype=w, device="cuda") for t in ("down", "up"))
    elif case["op"] == "policy":
        answered(case, s, g)
        n = case["n"]
        s["old"] = s["lp"] + 0.15 * normal(n, g=g)  # drawn a few steps ago
        s["reference"] = s["lp"] + 0.5 * normal(n, g=g)
        s["advantages"] = normal(n, g=g)
        s["weights"] = (0.5 + uniform(n, g=g)) / n
    elif case["op"] == "preference":
        answered(case, s, g)
        n, two = case["n"], 2 * case["pairs"]
        used = n - n // 16  # rows behind the last sequence fill the batch
        cut = torch.randint(0, used + 1, (two - 1,), generator=g, device="cuda").sort().values
        ends = torch.tensor([0, used], device="cuda")
        s["starts"] = torch.cat((ends[:1], cut, ends[1:])).to(torch.int32)
        lp = torch.cat((ends[:1].double(), torch.where(s["tokens"] >= 0, s["lp"], 0.0).double().cumsum(0)))
        lp = lp[s["starts"][1:].long()] - lp[s["starts"][:-1].long()]
        length = s["starts"][1:] - s["starts"][:-1]
        s["reference"] = (lp + normal(two, g=g) * length.sqrt() * 2.0).float()
    else:
        found, total = places(case)
        inside = torch.zeros(total, dtype=torch.bool, device="cuda")
        for size, at in found:
            inside[at:at + size] = True
        w = TYPES[case["parameters"]]
        size = torch.exp(normal(total, g=g)) * 1e-3 * inside  # of an element's gradients
        s["flat"] = (normal(total, g=g) * 0.02 * inside).to(w)
        s["slopes"] = (normal(total, g=g) * size).to(w)
        s["first"], s["second"] = normal(total, g=g) * size * 0.3, size * size * (0.7 + 0.6 * uniform(total, g=g))
        s["scales"] = None
        if case["bits"] == 8:  # the second state as its root
            held, s["scales"] = [], []
            for state in (s["first"], s["second"].sqrt()):
                most = state.view(-1, BLOCK).abs().amax(1)
                scale = torch.exp2(torch.ceil(torch.log2(most.clamp(min=2.0 ** -90) / 448.0)))
                held.append((state.view(-1, BLOCK) / scale[:, None]).to(E4M3).view(-1))
                s["scales"].append(scale)
            s["first"], s["second"] = held
        s["steps"], s["found"] = 100, found
        s["views"] = {t: [s[t][at:at + size] for size, at in found] for t in ("flat", "slopes", "first", "second")}
        if s["scales"]:
            for t, scale in zip(("first_scales", "second_scales"), s["scales"]):
                s["views"][t] = [scale[at // BLOCK:-(-(at + size) // BLOCK)] for size, at in found]
    return s


# ----------------------------------------------------------------------------- plain forms
def floats_of(s):
    """Clause outputs (n, c) in float32."""
    if s["x"] != "bits":
        return s["x_in"].float()
    at = torch.arange(32, dtype=torch.int32, device="cuda")
    return ((s["x_in"][:, :, None] >> at) & 1).view(s["n"], -1)[:, :s["c"]].float()


def of_own(s, value):
    """(n, m r): each row's r values in its adapter's place, zeros elsewhere."""
    mine = torch.arange(s["m"], device="cuda")[None, :] == s["which"][:, None]
    return (value[:, None, :] * mine[:, :, None]).view(s["n"], -1)


def own_of(s, every):
    """(n, r): of each row's values for all adapters those of its own."""
    at = s["which"].clamp(min=0).long()[:, None, None].expand(-1, 1, s["r"])
    return every.view(s["n"], s["m"], s["r"]).gather(1, at)[:, 0] * (s["which"] >= 0)[:, None]


def plain_adapt(s):
    m, r = s["m"], s["r"]
    hidden = own_of(s, floats_of(s) @ s["down"].float().view(m * r, -1).t())
    up = s["up"].float().permute(0, 2, 1).reshape(m * r, -1)
    return s["in"].float() + SCALE * (of_own(s, hidden) @ up), hidden


def plain_gradient(s):
    m, r, w = s["m"], s["r"], TYPES[s["weights"]]
    grad = s["in"].float() * SCALE
    d_up = (of_own(s, s["hidden"]).t() @ grad).view(m, r, -1).permute(0, 2, 1)
    back = own_of(s, grad @ s["up"].float().permute(1, 0, 2).reshape(-1, m * r))
    d_down = (of_own(s, back).t() @ floats_of(s)).view(m, r, -1)
    return d_down.to(w), d_up.to(w)


def log_probabilities(s):
    """(log probability of each row's answer, 0 where there is none; all answers' probabilities)"""
    z = s["in"].float()
    if s["temperature"] is not None:
        z = z / s["temperature"][:, None]
    z = z - z.amax(1, keepdim=True)
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    lp = z.gather(1, s["tokens"].clamp(min=0).long()[:, None])[:, 0] - torch.log(total[:, 0])
    return torch.where(s["tokens"] >= 0, lp, 0.0), p / total


def slopes(s, p, c):
    """The scores' gradient where c is that of the rows' log probabilities."""
    c = torch.where(s["tokens"] >= 0, c, 0.0)
    if s["temperature"] is not None:
        c = c / s["temperature"]
    grad = -c[:, None] * p
    grad.scatter_add_(1, s["tokens"].clamp(min=0).long()[:, None], c[:, None])
    return grad.to(TYPES[s["out"]])


def plain_policy(s):
    lp, p = log_probabilities(s)
    a, w, far = s["advantages"], s["weights"], s["reference"] - lp
    ratio = torch.exp(lp - s["old"])
    free, held = ratio * a, ratio.clamp(1.0 - CLIP, 1.0 + CLIP) * a
    loss = w * (KL * (torch.expm1(far) - far) - torch.minimum(free, held))
    c = w * (-KL * torch.expm1(far) - torch.where(free <= held, free, 0.0))
    none = s["tokens"] < 0
    return torch.where(none, 0.0, loss), slopes(s, p, c), lp


def plain_preference(s):
    lp, p = log_probabilities(s)
    pairs = s["pairs"]
    row = torch.arange(s["n"], device="cuda")
    mine = ((row >= s["starts"][:-1, None]) & (row < s["starts"][1:, None])).float()  # sequences x rows
    said = (mine * lp).sum(1)
    margin = BETA * (said - s["reference"]).view(pairs, 2)
    margin = margin[:, 0] - margin[:, 1]
    softplus = torch.clamp(margin, min=0.0) + torch.log1p(torch.exp(-margin.abs()))  # log(1 + exp(margin))
    loss = (softplus - (1.0 - SMOOTHING) * margin) / pairs
    c = (1.0 / (1.0 + torch.exp(-margin)) - (1.0 - SMOOTHING)) * (BETA / pairs)
    c = torch.stack((c, -c), 1).view(-1, 1)
    return loss, slopes(s, p, (mine * c).sum(0)), said


def mixed(h):
    """32 bits from 32 bits, in int64."""
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def chances(steps, count):
    """For each element (its place counts each tensor before it as a multiple of 256 long) three numbers of
    16 bits over 2^16: for the first and second state and for the parameter."""
    key = mixed(mixed(torch.tensor(steps, device="cuda")) ^ 0)  # the seed is 0
    a = mixed(torch.arange(count, device="cuda") ^ key)
    b = (a * 0x9E3779B9) & 0xFFFFFFFF
    return [(v.float() / 65536.0) for v in (a & 0xFFFF, a >> 16, b >> 16)]


def steps_of(size, fraction, least):
    """The distance of numbers of `fraction` bits and at least 2^least at `size`."""
    e = torch.frexp(size)[1] - 1
    return torch.ldexp(torch.ones_like(size), e.clamp(min=least) - fraction)


def drawn_to(x, chance, fraction, least):
    """x rounded up or down to a number of so many bits, to the nearer one more often."""
    step = steps_of(x.abs(), fraction, least)
    return torch.copysign(torch.floor(x.abs() / step + chance) * step, x)


def block_scales(size):
    most = size.view(-1, BLOCK).amax(1)
    bits = (most.view(torch.int32) + 0x1FFFFF) >> 23  # 1.75 * 2^e is the largest that 2^(e - 8) holds
    return torch.ldexp(torch.ones_like(most), bits.clamp(min=37) - 135)


def plain_adamw(s):
    s["steps"] += 1
    total, w = s["flat"].numel(), TYPES[s["parameters"]]
    first, second = s["first"].float(), s["second"].float()
    if s["bits"] == 8:
        first, second = [(x.view(-1, BLOCK) * y[:, None]).view(-1) for x, y in zip((first, second), s["scales"])]
        second = second * second
    g, p = s["slopes"].float(), s["flat"].float()
    first = BETAS[0] * first + (1.0 - BETAS[0]) * g
    second = BETAS[1] * second + (1.0 - BETAS[1]) * (g * g)
    root = torch.sqrt(second)
    rate = LR / (1.0 - BETAS[0] ** s["steps"])
    p = p * (1.0 - LR * DECAY) - rate * first / (root * (1.0 / math.sqrt(1.0 - BETAS[1] ** s["steps"])) + EPS)
    if s["bits"] == 8 or s["parameters"] != "float32":
        chance = chances(s["steps"], total)
    if s["parameters"] != "float32":
        p = drawn_to(p, chance[2], *((10, -14) if s["parameters"] == "float16" else (7, -126)))
    s["flat"].copy_(p.to(w))
    if s["bits"] == 32:
        s["first"].copy_(first)
        s["second"].copy_(second)
        return s["flat"], s["first"], s["second"]
    scale = block_scales(first.abs())
    x = (first.view(-1, BLOCK) / scale[:, None]).view(-1)
    s["first"].copy_(drawn_to(x, chance[0], 3, -6).to(E4M3))
    s["scales"][0].copy_(scale)
    scale = block_scales(root)
    x = (root.view(-1, BLOCK) / scale[:, None]).view(-1)
    step = steps_of(x, 3, -6)
    low = torch.floor(x / step) * step
    high = low + step
    # up with the chance that keeps the square's mean; what is not zero stays so
    up = (x * x - low * low > chance[1] * (high * high - low * low)) | ((low == 0.0) & (x > 0.0))
    s["second"].copy_(torch.where(up, high, low).to(E4M3))
    s["scales"][1].copy_(scale)
    return s["flat"], s["first"], s["second"], s["scales"]


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"adapt": plain_adapt, "gradient": plain_gradient, "policy": plain_policy,
                "preference": plain_preference, "adamw": plain_adamw}[op](s)
    from ytm_amd import tune

    if op == "adapt":
        hidden = torch.empty(s["n"], s["r"], device="cuda")
        return tune.adapt(s["in"], s["x_in"], s["down"], s["up"], s["which"], scale=SCALE, hidden=hidden,
                          out=s["to"]), hidden
    if op == "gradient":
        return tune.adapt_gradient(s["in"], s["x_in"], s["down"], s["up"], s["which"], s["hidden"], scale=SCALE,
                                   out=s["to"])
    if op == "policy":
        return tune.policy_loss(s["in"], s["tokens"], s["old"], s["advantages"], reference=s["reference"], kl=KL,
                                clip=CLIP, weights=s["weights"], temperature=s["temperature"], out=s["to"])
    if op == "preference":
        return tune.preference_loss(s["in"], s["tokens"], s["starts"], s["reference"], beta=BETA,
                                    smoothing=SMOOTHING, temperature=s["temperature"], out=s["to"])
    if "plan" not in s:  # made once, as a program that teaches makes it
        v = s["views"]
        held = {t: v[t] for t in ("first", "second", "first_scales", "second_scales") if t in v}
        s["plan"] = tune.AdamW(v["flat"], v["slopes"], bits=s["bits"], states=held, steps=s["steps"], seed=0)
    s["plan"].step(lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY)
    return (s["flat"], s["first"], s["second"]) + ((s["scales"],) if s["bits"] == 8 else ())


# ------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op in ("adapt", "gradient"):
        n, c, k, r = case["n"], case["c"], case["k"], case["r"]
        x = n * (-(-c // 32) * 4 if case["x"] == "bits" else c * SIZE[case["x"]])
        w, scores = SIZE[case["weights"]], n * k * SIZE[case["scores"]]
        met = min(n, case["m"])  # adapters that rows name, at most
        if op == "adapt":
            return {"bytes": x + scores + n * k * 4 + met * r * (c + k) * w + n * r * 4, "flops": 2.0 * n * r * (c + k)}
        return {"bytes": x + scores + n * r * 4 + met * r * k * w + case["m"] * r * (c + k) * w,
                "flops": 2.0 * n * r * (c + 2 * k)}
    if op == "adamw":
        size, w = sum(size for size, _ in places(case)[0]), SIZE[case["parameters"]]
        state = 4 if case["bits"] == 32 else 1 + 4 / BLOCK
        return {"bytes": size * (3 * w + 4 * state), "flops": 15.0 * size}
    return {"bytes": case["n"] * case["v"] * (SIZE[case["scores"]] + SIZE[case["out"]]),
            "flops": 6.0 * case["n"] * case["v"]}


# ----------------------------------------------------------------------------------- exact
def exact_rounding(x, chance, code):
    """The two neighbours of x >= 0 among numbers of `code`'s bits."""
    fraction, least = code
    e = torch.floor(torch.log2(torch.where(x > 0, x, 1.0)))
    step = torch.exp2(torch.where(x > 0, e, float(least)).clamp(min=least) - fraction)
    low = torch.floor(x / step) * step
    return low, low + step, (x - low) / step > 1.0 - chance


def exact(case, seed):
    """run()'s result from the definitions, in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    if op in ("adapt", "gradient"):
        n, c = case["n"], case["c"]
        if case["x"] == "bits":
            at = torch.arange(c, device="cuda")
            x = ((s["x_in"][:, at // 32].long() >> (at % 32)) % 2).double()
        else:
            x = s["x_in"].double()
        if op == "adapt":
            out, hidden = s["in"].double(), torch.zeros(n, case["r"], dtype=torch.float64, device="cuda")
            for a in range(case["m"]):
                rows = (s["which"] == a).nonzero()[:, 0]
                hidden[rows] = x[rows] @ s["down"][a].double().t()
                out[rows] += SCALE * (hidden[rows] @ s["up"][a].double().t())
            return out, hidden
        d_down, d_up = s["down"].double().zero_(), s["up"].double().zero_()
        for a in range(case["m"]):
            rows = (s["which"] == a).nonzero()[:, 0]
            grad = SCALE * s["in"][rows].double()
            d_up[a] = grad.t().contiguous() @ s["hidden"][rows].double()
            d_down[a] = (grad @ s["up"][a].double()).t().contiguous() @ x[rows]
        return d_down, d_up
    if op in ("policy", "preference"):
        t = s["tokens"].long()
        there = t >= 0
        z = s["in"].double()
        heat = torch.ones_like(t, dtype=torch.float64) if s["temperature"] is None else s["temperature"].double()
        log = torch.log_softmax(z / heat[:, None], 1)
        row = torch.arange(case["n"], device="cuda")
        lp = torch.where(there, log[row, t.clamp(min=0)], 0.0)
        if op == "policy":
            ratio, a, w = torch.exp(lp - s["old"].double()), s["advantages"].double(), s["weights"].double()
            gap = s["reference"].double() - lp
            bounded = torch.where(a > 0, ratio.clamp(max=1 + CLIP), ratio.clamp(min=1 - CLIP))
            said, loss = lp, there * w * (KL * (torch.exp(gap) - gap - 1) - bounded * a)
            c = w * (KL * (1 - torch.exp(gap)) - a * ratio * (bounded == ratio))
        else:
            pairs, starts = case["pairs"], s["starts"].long()
            of = torch.searchsorted(starts, row, right=True) - 1  # the last sequence that begins at or before
            of = torch.where(row < starts[-1], of, 2 * pairs)
            said = torch.zeros(2 * pairs + 1, dtype=torch.float64, device="cuda").index_add_(0, of, lp)[:-1]
            lead = said - s["reference"].double()
            lead = BETA * (lead[0::2] - lead[1::2])
            won = torch.sigmoid(lead)
            loss = -((1 - SMOOTHING) * torch.log(won) + SMOOTHING * torch.log1p(-won)) / pairs
            up = (won - 1 + SMOOTHING) * BETA / pairs
            c = torch.cat((torch.stack((up, -up), 1).view(-1), torch.zeros(1, device="cuda", dtype=torch.float64)))[of]
        c = there * c / heat
        grad = torch.exp(log).mul_(-c[:, None])
        grad[row, t.clamp(min=0)] += c
        return loss, grad, said
    k = s["steps"] + 1
    m, v = s["first"].double(), s["second"].double()
    if case["bits"] == 8:
        m *= s["scales"][0].double().repeat_interleave(BLOCK)
        v = (v * s["scales"][1].double().repeat_interleave(BLOCK)) ** 2
    g, p = s["slopes"].double(), s["flat"].double()
    m = BETAS[0] * m + (1 - BETAS[0]) * g
    v = BETAS[1] * v + (1 - BETAS[1]) * g ** 2
    p -= LR * DECAY * p + LR * (m / (1 - BETAS[0] ** k)) / (torch.sqrt(v / (1 - BETAS[1] ** k)) + EPS)
    chance = [c.double() for c in chances(k, p.numel())]
    if case["parameters"] != "float32":
        low, high, up = exact_rounding(p.abs(), chance[2], (10, -14) if case["parameters"] == "float16" else (7, -126))
        p = torch.copysign(torch.where(up, high, low), p)
    if case["bits"] == 32:
        return p, m, v
    held, scales = [], []
    for state, c in ((m, chance[0]), (v.sqrt(), chance[1])):
        most = state.abs().view(-1, BLOCK).amax(1)
        scale = torch.exp2(torch.ceil(torch.log2(most.clamp(min=1.75 * 2.0 ** -90) / 448)))
        y = state.abs() / scale.repeat_interleave(BLOCK)
        low, high, up = exact_rounding(y, c, (3, -6))
        if len(held):
            up = ((y ** 2 - low ** 2) / (high ** 2 - low ** 2) > c) | ((low == 0) & (y > 0))
        held.append(torch.copysign(torch.where(up, high, low), state))
        scales.append(scale)
    return p, held[0], held[1], scales
