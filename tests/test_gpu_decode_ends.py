"""The answering operators at the ends of what their operands may be."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ytm_amd = pytest.importorskip("ytm_amd")
from ytm_amd import decode  # noqa: E402


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


# few answers, hundreds of them kept, thousands of equal ones, a row long enough to be sliced
LENGTHS = [4, 100, 3000, 20001, 40000]


def ties(V):
    """Two rows in which most of the answers are the best, answer 1 the first of them."""
    x = torch.zeros(2, V, device="cuda")
    x[:, 0] = -1.0
    x[1, V // 2:] = -3.0
    return x, torch.linspace(0, 2, V, device="cuda")  # noise that likes the last answers


@pytest.mark.parametrize("V", LENGTHS)
@pytest.mark.parametrize("kept", [2, 50, 200, 1000, 0])
def test_choose_top_p_not_a_number(V, kept):
    """No bound, as 1 is, however many answers the other filters leave."""
    x, noise = ties(V)
    x = x + torch.arange(V, device="cuda") % 7 * 0.125
    k = torch.full((2,), kept, dtype=torch.int32, device="cuda")
    m = torch.full((2,), 0.1, device="cuda")
    p = torch.full((2,), float("nan"), device="cuda")
    for more in ({}, {"min_p": m}):
        assert same(decode.choose(x, top_k=k, top_p=p, noise=noise, **more),
                    decode.choose(x, top_k=k, noise=noise, **more))


@pytest.mark.parametrize("V", LENGTHS)
@pytest.mark.parametrize("share", [1.0000001, 2.0, float("inf")])
def test_choose_min_p_above_one(V, share):
    """No answer reaches more than the best one's share: the first answer alone is kept."""
    x, noise = ties(V)
    for more in ({}, {"top_p": torch.full((2,), 0.9, device="cuda")},
                 {"top_k": torch.full((2,), 300, dtype=torch.int32, device="cuda")}):
        index, log = decode.choose(x, min_p=torch.full((2,), share, device="cuda"), noise=noise, **more)
        assert index.tolist() == [1, 1] and log.tolist() == [0.0, 0.0]
    index, _ = decode.choose(x, min_p=torch.ones(2, device="cuda"), noise=noise)  # all of the best ones
    assert index.tolist() == [V - 1, V // 2 - 1]


def test_choose_more_rows_than_a_launch_takes():
    N, V = (1 << 22) + 5, 3
    x = torch.randint(-8, 9, (N, V), device="cuda").float()
    index, log = decode.choose(x)
    best = torch.where(x == x.amax(1, keepdim=True), torch.arange(V, device="cuda"), V).amin(1)
    assert torch.equal(index.long(), best)
    assert bool(((log.double() - torch.log_softmax(x.double(), 1).amax(1)).abs() <= 2.0**-18).all())
    k = torch.ones(N, dtype=torch.int32, device="cuda")
    first, none = decode.choose(x, top_k=k)
    assert torch.equal(index, first) and not bool(none.any())


def test_readout_more_outputs_than_a_launch_takes():
    """65535 rows x 786433 outputs of float16."""
    N, C, K = 65535, 8, 786433
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("takes 103 GB of device memory")
    codes = torch.zeros(K, 16, dtype=torch.uint8, device="cuda")
    codes[:, :4] = torch.randint(0, 256, (K, 4), device="cuda", dtype=torch.uint8)
    x = torch.randint(-4, 5, (N, C), device="cuda").float()
    scales = torch.ones(K, 1, device="cuda")
    out = torch.empty(N, K, dtype=torch.float16, device="cuda")
    decode.readout(x, codes, scales, out=out)
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    w = values[torch.stack((codes[:, :4] & 15, codes[:, :4] >> 4), 2).view(K, C).int()].t().contiguous()
    wrong = sum(int((out[n:n + 1024] != (x[n:n + 1024] @ w).half()).any()) for n in range(0, N, 1024))
    del out
    torch.cuda.empty_cache()
    assert wrong == 0


@pytest.mark.parametrize("N", [1, 5, 40])
@pytest.mark.parametrize("C", [5, 300])
def test_readout_one_row_of_codes_or_scales_for_all(N, C):
    """Codes or scales that are the same for all outputs (stride 0) read as if they were copies."""
    K = 37
    codes = torch.randint(0, 256, (K, 16 * -(-C // 32)), device="cuda", dtype=torch.uint8)
    scales, x = torch.rand(K, -(-C // 32), device="cuda"), torch.randn(N, C, device="cuda")
    for c, s in ((codes[:1].expand(K, -1), scales), (codes, scales[:1].expand(K, -1)),
                 (codes[:1].expand(K, -1), scales[:1].expand(K, -1))):
        assert torch.equal(decode.readout(x, c, s), decode.readout(x, c.contiguous(), s.contiguous()))


def test_written_tensors_are_known_to_autograd():
    """What a backward pass has kept is not used once an operator has written to it."""
    scores, w = torch.randn(3, 40, device="cuda"), torch.ones(3, 40, device="cuda", requires_grad=True)
    codes, scales = torch.full((40, 16), 0x22, dtype=torch.uint8, device="cuda"), torch.ones(40, 1, device="cuda")
    for write in (lambda out: decode.adjust_scores(scores, out=out),
                  lambda out: decode.readout(torch.ones(3, 32, device="cuda"), codes, scales, out=out)):
        kept = torch.randn(3, 40, device="cuda")
        y = (w * kept).sum()
        write(kept)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_written_between_what_is_read():
    """Rows of the output that lie between rows of an input are no overlap; a part of the scores is."""
    N, V = 6, 100
    want = torch.randn(N, V, device="cuda")
    bias = torch.randn(V, device="cuda")
    both = torch.zeros(N, 2 * V, device="cuda")
    both[:, :V] = want
    decode.adjust_scores(both[:, :V], bias=bias, out=both[:, V:])
    assert torch.equal(both, torch.cat((want, want + bias), 1))
    x, ones = torch.ones(N, 32, device="cuda"), torch.ones(V, 1, device="cuda")
    both = torch.ones(N, 32 + V, device="cuda")
    codes = torch.full((V, 16), 0x22, dtype=torch.uint8, device="cuda")
    decode.readout(both[:, :32], codes, ones, out=both[:, 32:])
    assert torch.equal(both, torch.cat((x, 32 * torch.ones(N, V, device="cuda")), 1))
    half = torch.randn(N, 2 * V, device="cuda").half()
    want = half[:, :V].bfloat16() + bias.bfloat16().float()  # in place, from one type of 16 bits to another
    scores = half.view(torch.bfloat16)
    scores[:, :V] = half[:, :V].bfloat16()
    decode.adjust_scores(scores[:, :V], bias=bias.bfloat16().float(), out=half[:, :V])
    assert torch.equal(half[:, :V], want.half())
    big = torch.randn(2 * N, V, device="cuda")
    for out in (big[1:N + 1], big.as_strided((N, V), (V, 1), 3), big.view(torch.float16)[:N, :V]):
        with pytest.raises(ValueError, match="overlaps"):
            decode.adjust_scores(big[:N], bias=bias, out=out)


@pytest.mark.parametrize("N", [1, 20])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype,least", [("float16", -24), ("bfloat16", -133), ("float32", -133)])
def test_readout_least_values(dtype, least, group, N):
    """Rows' subnormal values count; of float32 those down to the least of bfloat16."""
    at = torch.arange(least, least + 24)
    x = torch.zeros(N, 128, dtype=torch.float64)
    x[:, torch.arange(24) * 5] = torch.exp2(at.double())
    codes = torch.full((3, 64), 0x22, dtype=torch.uint8, device="cuda")
    scales = torch.full((3, 128 // group), 2.0 ** (100 if least < -100 else 0), device="cuda")
    got = decode.readout(x.to(getattr(torch, dtype)).cuda(), codes, scales, group=group)
    want = torch.exp2(at.double()).sum() * scales[0, 0].item()  # 24 bits
    assert bool((got.double().cpu() == want).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(1, 50), (7, 9001)])
def test_adjust_over_the_bias(N, V, dtype):
    scores, bias = torch.randn(N, V, device="cuda").to(dtype), torch.randn(N, V, device="cuda")
    want = scores.float() + bias
    assert decode.adjust_scores(scores, bias=bias, out=bias) is bias
    assert torch.equal(bias, want)
