"""Cases for timing the operators that answer with words: the 4-bit readout of clause outputs,
the shaping of scores by history, bias and grammar, and the choice of an answer.

Each case is one call as a program that answers step by step makes it.  With `own` false the
operators are computed in their plain form, elementary torch operations in float32; with `own`
true by ytm_amd.decode.  Models' sizes are those of the benchmark configurations (2000 to 20000
clauses, 10 classes, 10000 words); larger answer sets and batches are generic.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
LARGEST = torch.finfo(torch.float32).max


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one image's class scores from the 2000 clauses of the flat image model: latency
        dict(name="readout_digits", op="readout", n=1, c=2000, k=10, x="bits", group=32, scale="float32",
             out="float32"),
        # the next word of one text: 10000 clauses, 10000 words; the weights' bytes
        dict(name="readout_word", op="readout", n=1, c=10000, k=10000, x="bits", group=64, scale="float16",
             out="float32"),
        # a few texts at once, clause outputs averaged over models (no longer bits), an odd number of words
        dict(name="readout_averages", op="readout", n=13, c=8000, k=10007, x="float32", group=32, scale="float32",
             out="float32"),
        # a server's batch over a large vocabulary, a clause count no tile divides
        dict(name="readout_batch", op="readout", n=96, c=9973, k=32001, x="float16", group=128, scale="float16",
             out="float16"),
        # a set of documents at once, the largest clause count
        dict(name="readout_documents", op="readout", n=512, c=20000, k=10000, x="bfloat16", group=128,
             scale="bfloat16", out="float32"),
        # one text of at most 150 words, penalties alone: latency
        dict(name="adjust_one", op="adjust", n=1, v=10000, t=150, x="float32", out="float32", bias="none",
             allowed="none"),
        # a server's batch under grammars, with a bias for all, an odd number of words
        dict(name="adjust_grammar", op="adjust", n=64, v=32001, t=2048, x="bfloat16", out="float32", bias="shared",
             allowed="rows"),
        # the largest batch and vocabulary, long histories
        dict(name="adjust_many", op="adjust", n=256, v=131072, t=4096, x="float32", out="float32", bias="shared",
             allowed="rows"),
        # the likeliest word of one text: latency
        dict(name="choose_best", op="choose", n=1, v=10000, x="float32", noise=False, filters="none"),
        # a drawn word of one text, large vocabulary, all filters
        dict(name="choose_one", op="choose", n=1, v=131072, x="float32", noise=True, filters="all"),
        # a server's batch, 16-bit scores, all filters, an odd number of words
        dict(name="choose_rows", op="choose", n=64, v=32001, x="bfloat16", noise=True, filters="all"),
        # the largest batch and vocabulary
        dict(name="choose_many", op="choose", n=256, v=131072, x="float32", noise=True, filters="all"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["readout", "readout", "adjust", "choose"])
    if op == "readout":
        n, c, k = log(1, 512), log(200, 20000), log(10, 32768)
        k = min(k, 3 * 10 ** 8 // c)
        n = max(1, min(n, 10 ** 11 // (c * k)))
        x = rng.choice(["bits", "float32", "float16", "bfloat16"])
        out = "float32" if x == "bits" else rng.choice(["float32", x])
        return dict(op=op, n=n, c=c, k=k, x=x, group=rng.choice([32, 64, 128, 256]),
                    scale=rng.choice(["float32", "float16", "bfloat16"]), out=out)
    n, v, x = log(1, 256), log(100, 131072), rng.choice(["float32", "float16", "bfloat16"])
    if op == "adjust":
        return dict(op=op, n=n, v=v, t=log(1, 4096), x=x, out=rng.choice(["float32", x]),
                    bias=rng.choice(["none", "shared", "rows"]), allowed=rng.choice(["none", "shared", "rows"]))
    return dict(op=op, n=n, v=v, x=x, noise=rng.random() < 0.8, filters=rng.choice(["none", "k", "p", "min", "all"]))


# ---------------------------------------------------------------------------------- inputs
def zipf(shape, v, g):
    """Words drawn like words in text: the r-th most common about 1 / r as often."""
    return (v ** torch.rand(shape, generator=g, device="cuda") - 1).to(torch.int32).clamp_(0, v - 1)


def weights(c, k, group, scale, g):
    """Clause weights as training leaves them (whole numbers around zero), held in 4 bits: codes
    (k, 16 ceil(c / 32)) bytes, the even clause in the low half, and a scale per group."""
    per, padded = -(-c // group), 32 * -(-c // 32)
    w = (torch.randn(k, per * group, generator=g, device="cuda") * 8.0).round_()
    w[:, c:] = 0.0
    w = w.view(k, per, group)
    s = (w.abs().amax(2) / 6.0).clamp_(min=1e-3).to(TYPES[scale])
    w = (w / s.float()[:, :, None]).view(k, per * group)[:, :padded]
    middle = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    code = torch.bucketize(w.abs(), middle, out_int32=True).to(torch.uint8)
    code |= (w < 0).to(torch.uint8) << 3
    return (code[:, 0::2] | code[:, 1::2] << 4).contiguous(), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "readout":
        n, c, k = case["n"], case["c"], case["k"]
        s["codes"], s["scales"] = weights(c, k, case["group"], case["scale"], g)
        if case["x"] == "bits":  # a tenth of the clauses fire
            words = torch.zeros(n, -(-c // 32), dtype=torch.int64, device="cuda")
            for b in range(32):
                words |= (torch.rand(words.shape, generator=g, device="cuda") < 0.1).long() << b
            if c % 32:
                words[:, -1] &= (1 << c % 32) - 1
            s["in"] = (words - (words >> 31 << 32)).to(torch.int32)
        else:  # shares of models or patches in which a clause fires, most of them zero
            x = torch.rand(n, c, generator=g, device="cuda")
            s["in"] = torch.where(x < 0.3, torch.rand(n, c, generator=g, device="cuda"), 0.0).to(TYPES[case["x"]])
        s["to"] = torch.empty(n, k, dtype=TYPES[case["out"]], device="cuda")
        return s
    n, v = case["n"], case["v"]
    # scores as a readout gives them: whole rows around zero, a few words far above
    x = torch.randn(n, v, generator=g, device="cuda") * 3.0
    x += 6.0 * (torch.rand(n, v, generator=g, device="cuda") < 20.0 / v)
    x = x.to(TYPES[case["x"]])
    if case["op"] == "adjust":
        t = case["t"]
        s["in"] = x
        s["to"] = torch.empty(n, v, dtype=TYPES[case["out"]], device="cuda")
        s["tokens"] = zipf((n, t), v, g)
        s["lengths"] = torch.randint(0, t + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["prompt"] = (s["lengths"] * torch.rand(n, generator=g, device="cuda")).to(torch.int32)
        s["repetition"] = 1.0 + 0.3 * torch.rand(n, generator=g, device="cuda")
        s["frequency"] = 0.5 * torch.rand(n, generator=g, device="cuda")
        s["presence"] = torch.rand(n, generator=g, device="cuda") - 0.2
        s["bias"] = s["allowed"] = None
        if case["bias"] != "none":  # a few words wanted or not
            shape = (v,) if case["bias"] == "shared" else (n, v)
            s["bias"] = torch.randn(shape, generator=g, device="cuda") * (torch.rand(shape, generator=g, device="cuda") < 0.05)
        if case["allowed"] != "none":  # a grammar's words: from a few to nearly all of them
            rows = 1 if case["allowed"] == "shared" else n
            share = torch.rand(rows, 1, generator=g, device="cuda") ** 3
            words = torch.zeros(rows, -(-v // 32), dtype=torch.int64, device="cuda")
            for b in range(32):
                words |= (torch.rand(words.shape, generator=g, device="cuda") < share).long() << b
            words = (words - (words >> 31 << 32)).to(torch.int32)
            s["allowed"] = words[0].contiguous() if case["allowed"] == "shared" else words
        return s
    # a grammar has left out a third of the words
    s["in"] = x.masked_fill_(torch.rand(n, v, generator=g, device="cuda") < 0.33, -math.inf)
    f = case["filters"]
    s["temperature"] = s["k"] = s["p"] = s["min"] = s["noise"] = None
    if f != "none" or case["noise"]:
        s["temperature"] = 0.5 + torch.rand(n, generator=g, device="cuda")
        if n > 4:
            s["temperature"][n // 2] = 0.0  # one row wants its best word
    if f in ("k", "all"):  # one row in four has no bound
        k = (5.0 * 40.0 ** torch.rand(n, generator=g, device="cuda")).to(torch.int32)
        s["k"] = torch.where(torch.rand(n, generator=g, device="cuda") < (0.25 if n > 1 else 0.0), 0, k).to(torch.int32)
    if f in ("p", "all"):
        s["p"] = 0.8 + 0.19 * torch.rand(n, generator=g, device="cuda")
    if f in ("min", "all"):
        s["min"] = 0.05 * torch.rand(n, generator=g, device="cuda")
    if case["noise"]:
        u = torch.rand(n, v, generator=g, device="cuda").clamp_(1e-7, 1.0 - 1e-7)
        s["noise"] = -torch.log(-torch.log(u))
    return s


# ----------------------------------------------------------------------------- plain forms
def bits_of(words, count):
    """The bits of int32 words, least significant first, (rows, count)."""
    at = torch.arange(32, dtype=torch.int32, device=words.device)
    return ((words[:, :, None] >> at) & 1).view(words.shape[0], -1)[:, :count]


def plain_readout(s):
    codes, c, group = s["codes"], s["c"], s["group"]
    value = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=codes.device)
    w = value[torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], -1)[:, :c].int()]
    w = w * s["scales"].float().repeat_interleave(group, 1)[:, :c]
    x = bits_of(s["in"], c).float() if s["x"] == "bits" else s["in"].float()
    return (x @ w.t()).to(TYPES[s["out"]])


def plain_adjust(s):
    x = s["in"].float()
    n, v = x.shape
    at = torch.arange(s["t"], device=x.device)[None, :]
    told, answered = at < s["lengths"][:, None], at >= s["prompt"][:, None]
    tokens = s["tokens"].long()
    every = torch.zeros(n, v, device=x.device).scatter_add_(1, tokens, told.float())
    count = torch.zeros(n, v, device=x.device).scatter_add_(1, tokens, (told & answered).float())
    r = s["repetition"][:, None]
    x = torch.where(every > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0).float()
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        words = s["allowed"] if s["allowed"].dim() == 2 else s["allowed"][None, :]
        x = torch.where(bits_of(words, v) > 0, x, -math.inf)
    return x.to(TYPES[s["out"]])


def plain_choose(s):
    z = s["in"].float()
    n, v = z.shape
    first = torch.zeros(n, 1, dtype=torch.bool, device=z.device)
    if s["temperature"] is not None:
        t = s["temperature"][:, None]
        first = t <= 0
        z = z / torch.where(first, 1.0, t)
    z = torch.nan_to_num(z, nan=-math.inf, posinf=LARGEST, neginf=-math.inf)
    z, order = torch.sort(z, dim=1, descending=True, stable=True)
    best, at = z[:, :1], torch.arange(v, device=z.device)[None, :]
    keep = z > -math.inf
    if s["min"] is not None:
        keep = keep & (z >= best + torch.log(s["min"])[:, None])
    if s["k"] is not None:
        k = s["k"][:, None]
        keep = keep & ((at < k) | (k <= 0))
    keep = keep & ((at == 0) | ~first)
    if s["p"] is not None:
        mass = torch.where(keep, torch.exp(z - best), 0.0)
        before = torch.cumsum(mass, 1) - mass
        keep = keep & ((at == 0) | (before < s["p"][:, None] * mass.sum(1, keepdim=True)))
    total = torch.where(keep, torch.exp(z - best), 0.0).sum(1)
    z = torch.empty_like(z).scatter_(1, order, z)
    keep = torch.empty_like(keep).scatter_(1, order, keep)
    y = z if s["noise"] is None else z + s["noise"]
    token = torch.where(keep, y.clamp(min=-LARGEST), -math.inf).argmax(1)
    log = z.gather(1, token[:, None])[:, 0] - best[:, 0] - torch.log(total)
    none = best[:, 0] == -math.inf
    return torch.where(none, -1, token).to(torch.int32), torch.where(none, -math.inf, log)


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"readout": plain_readout, "adjust": plain_adjust, "choose": plain_choose}[op](s)
    from ytm_amd import decode

    if op == "readout":
        return decode.readout(s["in"], s["codes"], s["scales"], group=s["group"], clauses=s["c"], out=s["to"])
    if op == "adjust":
        return decode.adjust_scores(s["in"], tokens=s["tokens"], lengths=s["lengths"], prompt=s["prompt"],
                                    repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                                    bias=s["bias"], allowed=s["allowed"], out=s["to"])
    return decode.choose(s["in"], temperature=s["temperature"], top_k=s["k"], top_p=s["p"], min_p=s["min"],
                         noise=s["noise"])


# ------------------------------------------------------------------------------------ work
def work(case):
    n = case["n"]
    if case["op"] == "readout":
        c, k = case["c"], case["k"]
        x = -(-c // 32) * 4 if case["x"] == "bits" else c * SIZE[case["x"]]
        held = c / 2 + -(-c // case["group"]) * SIZE[case["scale"]]
        return {"bytes": k * held + n * x + n * k * SIZE[case["out"]], "flops": 2.0 * n * c * k}
    v = case["v"]
    if case["op"] == "adjust":
        rows = {"none": 0, "shared": 1, "rows": n}
        moved = n * v * (SIZE[case["x"]] + SIZE[case["out"]]) + 2 * n * case["t"]  # half of the histories
        return {"bytes": moved + 4 * rows[case["bias"]] * v + rows[case["allowed"]] * v / 8, "flops": 6.0 * n * v}
    return {"bytes": n * v * (SIZE[case["x"]] + (4 if case["noise"] else 0)) + 8 * n, "flops": 4.0 * n * v}


# ----------------------------------------------------------------------------------- exact
def exact(case, seed):
    """run()'s result from the definitions, in 64 bits."""
    s = prepare(case, seed)
    x = s["in"]
    if case["op"] == "readout":
        nibble = torch.empty(case["k"], 2 * s["codes"].shape[1], dtype=torch.uint8, device=x.device)
        nibble[:, 0::2], nibble[:, 1::2] = s["codes"] % 16, s["codes"] // 16
        nibble = nibble[:, :case["c"]]
        e, m = (nibble // 2 % 4).double(), (nibble % 2).double()  # E2M1: sign, two exponent bits, one of fraction
        w = torch.where(e == 0, m / 2, torch.exp2(e - 1) * (1 + m / 2)) * (1 - 2 * (nibble // 8).double())
        group = torch.arange(case["c"], device=x.device) // case["group"]
        w *= s["scales"].double()[:, group]
        if case["x"] == "bits":
            at = torch.arange(case["c"], device=x.device)
            x = (x[:, at // 32].long() >> (at % 32)) % 2
        return torch.matmul(w, x.double().t()).t()
    n, v = x.shape
    x = x.double()
    if case["op"] == "adjust":
        row = torch.arange(n, device=x.device)[:, None].expand(n, case["t"])
        at = torch.arange(case["t"], device=x.device).expand(n, case["t"])
        flat = (row * v + s["tokens"]).reshape(-1)
        told = (at < s["lengths"][:, None]).reshape(-1)
        answer = told & (at >= s["prompt"][:, None]).reshape(-1)
        every = torch.bincount(flat[told], minlength=n * v).view(n, v)
        count = torch.bincount(flat[answer], minlength=n * v).view(n, v)
        r = s["repetition"].double()[:, None].expand(n, v)
        factor = torch.where(every == 0, 1.0, torch.where(x > 0, 1 / r, r))
        x = x * factor - s["frequency"].double()[:, None] * count
        x -= s["presence"].double()[:, None] * count.clamp(max=1)
        if s["bias"] is not None:
            x = x + s["bias"].double()
        if s["allowed"] is not None:
            at = torch.arange(v, device=x.device)
            x[((s["allowed"].view(-1, -(-v // 32))[:, at // 32].long() >> (at % 32)) % 2 == 0).expand(n, v)] = -math.inf
        return x
    t = torch.ones(n, dtype=torch.float64, device=x.device) if s["temperature"] is None else s["temperature"].double()
    greedy = t <= 0
    x = x / torch.where(greedy, 1.0, t)[:, None]
    order = torch.argsort(-x, dim=1, stable=True)
    rank = torch.empty_like(order).scatter_(1, order, torch.arange(v, device=x.device).expand(n, v).contiguous())
    best = x.amax(1, keepdim=True)
    kept = x > -math.inf
    if s["min"] is not None:
        kept &= x >= best + s["min"].double().log()[:, None]
    if s["k"] is not None:
        kept &= rank < torch.where(s["k"] > 0, s["k"], v)[:, None]
    kept &= (rank == 0) | ~greedy[:, None]
    p = torch.softmax(torch.where(kept, x, -math.inf), 1)
    if s["p"] is not None:
        run_up = p.gather(1, order).cumsum(1).gather(1, rank) - p
        kept &= (rank == 0) | (run_up < s["p"].double()[:, None])
    y = x if s["noise"] is None else x + s["noise"].double()
    token = torch.where(kept, y, -math.inf).argmax(1)
    log = torch.log_softmax(torch.where(kept, x, -math.inf), 1).gather(1, token[:, None])[:, 0]
    return token.to(torch.int32), log
