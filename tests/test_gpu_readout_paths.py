"""The readout at sizes where its kernels run as they do in use: many chunks of clauses to a block,
many tiles of outputs, parts of a row's clauses.  Codes, scales and rows are random and every product
and sum is a whole number of 2^-3 below 2^21, which float32 holds: results have to be equal.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ytm_amd = pytest.importorskip("ytm_amd")
from ytm_amd import decode  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
VALUES = [0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6]


def check_exact(N, C, K, x, group, scale="f32"):
    g = torch.Generator(device="cuda").manual_seed(N + 7 * C + 13 * K + group)
    codes = torch.randint(0, 256, (K, 16 * -(-C // 32)), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.exp2(torch.randint(-2, 3, (K, -(-C // group)), generator=g, device="cuda").float())
    code = torch.stack((codes & 15, codes >> 4), 2).view(K, -1)[:, :C].int()
    w = torch.tensor(VALUES, dtype=torch.float64, device="cuda")[code]
    w *= scales.double().repeat_interleave(group, 1)[:, :C]
    if x == "bits":
        rows = torch.randint(-2**31, 2**31, (N, -(-C // 32)), generator=g, device="cuda").to(torch.int32)
        at = torch.arange(C, device="cuda")
        values = (rows[:, at // 32] >> (at % 32).int()) & 1
    else:
        rows = values = torch.randint(-4, 5, (N, C), generator=g, device="cuda").to(TYPES[x])
    want = values.double() @ w.t().contiguous()
    got = decode.readout(rows, codes, scales.to(TYPES[scale]), group=group, clauses=C)
    assert torch.equal(got.double(), want)


# 32, 64, 96 and 128 rows a block where rows are of 16 bits or bits; over 128 blocks, which are not cut
# into parts, of 6 (two groups of waves) or 12 pairs of chunks
@pytest.mark.parametrize("x", ["bits", "f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(20, 16501), (60, 16501), (90, 21001), (300, 10007)])
def test_many_rows_and_outputs(N, K, x, group):
    check_exact(N, 3001, K, x, group, "f16" if group == 64 else "f32")


@pytest.mark.parametrize("x", ["bits", "f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("N,C,K", [(300, 10000, 10007), (100, 20000, 13001), (20, 10000, 10007)])
def test_many_clauses(N, C, K, x, group):
    """40 to 79 pairs of chunks to a block; the last in parts of several pairs."""
    check_exact(N, C, K, x, group)


# parts of few rows: in blocks of 256 outputs and, where these are few, of 16
@pytest.mark.parametrize("x", ["bits", "f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("N,C,K", [(13, 8000, 10007), (16, 20000, 4001), (2, 20027, 1792), (1, 10000, 10007)])
def test_few_rows(N, C, K, x, group):
    check_exact(N, C, K, x, group, "bf16" if N == 13 else "f32")
