"""4-bit rows on the CPU: the format against rational arithmetic, the restatements, and what is refused."""

import math
from fractions import Fraction

import pytest
import torch

from research_b200.errors import KernelError
from research_b200.ops import quantized as q4

BF16 = torch.bfloat16


def rational_codes(values):
    """Codes, scale and least value of one group from the definition, in exact arithmetic (finite values, s > 0)."""

    least, most = min(values), max(values)
    # the quotient as a bf16: fp32 has 16 bits more than it, and a fifteenth of a sum of two bf16 is never that close to a tie
    s = torch.tensor(float(Fraction(most) - Fraction(least)) / 15.0, dtype=torch.float64).to(BF16).item()
    out = []
    for x in values:
        q = (Fraction(x) - Fraction(least)) / Fraction(s)
        out.append(min(15, round(q)))               # Python rounds a tie of a Fraction to the even number
    return out, s, least


def held_codes(rows, channels):
    """Codes in channel order, nibble by nibble from the documented layout."""

    codes = rows.codes.reshape(-1, rows.codes.shape[-1])
    width = codes.shape[1] * 2
    out = torch.empty(codes.shape[0], channels, dtype=torch.int64)
    for c in range(channels):
        word = c // 8 if width == 64 else c // 128 * 16 + 2 * (c % 64 // 8) + c // 64 % 2
        nibble = (c % 8) // 2 + 4 * (c % 2)
        out[:, c] = (codes[:, word * 4 + nibble // 2] >> (4 * (nibble % 2))) & 15
    return out


def tricky_groups():
    g = torch.Generator().manual_seed(3)
    groups = [torch.randn(64, generator=g), torch.randn(64, generator=g) * 1e-6, torch.randn(64, generator=g) * 1e30,
              torch.arange(64).float(),                                      # ties: s = 4.1875
              torch.arange(64).float() / 2,
              torch.cat([torch.tensor([0.0, 30.0]), torch.arange(62) * 1.0]),   # s = 4.125
              torch.cat([torch.tensor([-1.0, 29.0, 1e-9, -1e-9, 0.0]), torch.arange(59) * 0.5]),   # s = 2: ties but for 1e-9
              torch.randn(64, generator=g) * torch.logspace(-30, 3, 64),     # least and values 2^16 and more apart
              torch.randn(64, generator=g) + 1000.0,
              torch.cat([torch.tensor([-3.0, 27.0]), torch.tensor([1e-12, -1e-12, 1e-25, -1e-25, 0.0, -0.0]).repeat(10),
                         torch.tensor([2.0, 4.0])]),                     # ties but for 2^-40 and 2^-83 of the step
              torch.cat([torch.tensor([-105984.0]), torch.tensor([-9e-14, 9e-14] * 31), torch.tensor([32256.0])])]
    return [x.to(BF16) for x in groups]


@pytest.mark.parametrize("index", range(11))
def test_codes_are_the_nearest_in_exact_arithmetic(index):
    x = tricky_groups()[index]
    rows = q4.quantize_rows_q4(x)
    want, s, least = rational_codes([v.item() for v in x])
    assert held_codes(rows, 64)[0].tolist() == want
    assert rows.affine.flatten().tolist() == [s, least]


@pytest.mark.parametrize("channels,width", [(1, 64), (5, 64), (63, 64), (64, 64), (65, 128), (128, 128), (129, 256), (200, 256)])
def test_width_padding_and_layout(channels, width):
    g = torch.Generator().manual_seed(channels)
    x = torch.randn(3, 2, channels, generator=g).to(BF16)
    rows = q4.quantize_rows_q4(x)
    assert rows.codes.shape == (3, 2, width // 2) and rows.affine.shape == (3, 2, width // 64, 2)
    codes = held_codes(rows, channels).view(3, 2, channels)
    for first in range(0, width, 64):
        pair = rows.affine[..., first // 64, :].double()
        if first >= channels:
            assert pair.abs().sum() == 0
            continue
        part = x[..., first:first + 64].double()
        assert torch.equal(pair[..., 1], part.amin(-1))
        value = codes[..., first:first + 64].double() * pair[..., :1] + pair[..., 1:]
        # the nearest of 16 levels that reach from the least to the largest value, up to the rounding of the step
        assert ((value - part).abs() <= pair[..., :1] * (0.5 + 15 * 2 ** -8)).all()
        assert torch.equal(q4.dequantize_rows_q4(rows, channels, torch.float32)[..., first:first + 64], value.float())


def test_groups_without_spread_or_without_numbers():
    tiny = torch.finfo(BF16).tiny
    x = torch.zeros(7, 64, dtype=BF16)
    x[0] = 3.0
    x[1, 5] = math.nan
    x[2, 9] = math.inf
    x[3, 1] = -math.inf
    x[4, 0], x[4, 1] = 3e38, -3e38                       # a spread that fp32 does not have
    x[5, 0] = 14 * tiny                                  # s would be below the least normal number
    x[6, 0] = 15 * tiny
    back = q4.dequantize_rows_q4(q4.quantize_rows_q4(x), 64)
    assert torch.equal(back[0], x[0])
    assert back[1:5].isnan().all()
    assert torch.equal(back[5], torch.zeros(64, dtype=BF16))
    assert torch.equal(back[6], x[6])


def test_write_leaves_out_rows_outside_and_keeps_the_others():
    g = torch.Generator().manual_seed(0)
    B, T, H, D, pages, ps = 4, 5, 2, 64, 3, 4
    k, v = (torch.randn(B, T, H, D, generator=g).to(BF16) for _ in range(2))
    pools = [q4.empty_rows(B, pages, H, ps, channels=D) for _ in range(2)]
    for pool in pools:
        pool.codes.fill_(7)
        pool.affine.fill_(1.5)
    before = [q4.Q4Rows(*(t.clone() for t in pool)) for pool in pools]
    start = torch.tensor([0, 3, 10, -2])
    q4.kv_write_paged_q4(k, v, *pools, start)
    want = [q4.quantize_rows_q4(x) for x in (k, v)]
    for pool, old, held in zip(pools, before, want):
        for b in range(B):
            for r in range(pages * ps):
                t = r - int(start[b])
                for field in (0, 1):
                    now = pool[field][b, r // ps, :, r % ps]
                    assert torch.equal(now, held[field][b, t] if 0 <= t < T else old[field][b, r // ps, :, r % ps])
    back_k, back_v = q4.kv_read_paged_q4(*pools, T, start)
    inside = torch.tensor([[0 <= int(s) + t < pages * ps for t in range(T)] for s in start])
    for back, held in ((back_k, want[0]), (back_v, want[1])):
        assert torch.equal(back[inside], q4.dequantize_rows_q4(held, D)[inside])
        assert torch.count_nonzero(back[~inside]) == 0


@pytest.mark.parametrize("D,Hq,Hkv", [(16, 4, 2), (64, 3, 1), (128, 8, 8)])
def test_attention_restatement_against_a_loop(D, Hq, Hkv):
    g = torch.Generator().manual_seed(D)
    B, pages, ps = 5, 3, 5
    q = torch.randn(B, Hq, D, generator=g, dtype=torch.float64)
    pools = [q4.quantize_rows_q4(torch.randn(B, pages, Hkv, ps, D, generator=g)) for _ in range(2)]
    lengths, lo = torch.tensor([15, 40, 0, 4, 9]), torch.tensor([0, 11, 0, 4, -3])
    for pool in pools:                                   # masked rows hold what would spoil every sum
        pool.affine[3:, 2] = math.nan
    k, v = (q4.dequantize_rows_q4(pool, D, torch.float64).permute(0, 1, 3, 2, 4).reshape(B, pages * ps, Hkv, D) for pool in pools)
    got = q4.decode_attention_paged_q4(q, *pools, lengths, lo)
    for b in range(B):
        rows = slice(max(int(lo[b]), 0), min(int(lengths[b]), pages * ps))
        for h in range(Hq):
            if rows.start >= rows.stop:
                want = torch.zeros(D, dtype=torch.float64)
            else:
                p = torch.softmax(k[b, rows, h // (Hq // Hkv)] @ q[b, h] / math.sqrt(D), dim=0)
                want = p @ v[b, rows, h // (Hq // Hkv)]
            # fp32 sums of at most 15 rows and D channels: 150 roundings of 2^-24, of values up to 5
            torch.testing.assert_close(got[b, h * D:(h + 1) * D], want, atol=150 * 2 ** -24 * 5, rtol=0)


def test_linear_restatement():
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(2, 3, 70, generator=g, dtype=torch.float64), torch.randn(9, 70, generator=g)
    rows = q4.quantize_rows_q4(w)
    want = x @ q4.dequantize_rows_q4(rows, 70, torch.float64).t()
    torch.testing.assert_close(q4.linear_q4(x, rows), want, atol=70 * 2 ** -23 * 70, rtol=0)
    assert q4.linear_q4(x[:0], rows).shape == (0, 3, 9)


def _pools(B=2, pages=2, H=2, ps=4, D=64, device=None):
    return [q4.empty_rows(B, pages, H, ps, channels=D, device=device) for _ in range(2)]


def test_refusals_of_the_cache_calls():
    k = torch.zeros(2, 3, 2, 64, dtype=BF16)
    pools = _pools()
    for bad, words in [((k[0], k[0], *pools), "one shape and type"),
                       ((k, k.float(), *pools), "one shape and type"),
                       ((k.int(), k.int(), *pools), "one shape and type"),
                       ((k, k[:, :2], *pools), "one shape and type"),
                       ((k[:1], k[:1], *pools), "does not hold 1 sequences"),
                       ((k[:, :, :1], k[:, :, :1], *pools), "of 1 heads"),
                       ((k[..., :32].contiguous(), k[..., :32].contiguous(), *_pools(D=128)), "rows of 32 channels"),
                       ((k, k, pools[0], _pools(ps=8)[1]), "must have one shape"),
                       ((k, k, q4.Q4Rows(pools[0].codes[:, :1], pools[0].affine[:, :1]), pools[1]), "contiguous"),
                       ((k, k, q4.Q4Rows(pools[0].codes.int(), pools[0].affine), pools[1]), "uint8 codes"),
                       ((k, k, q4.Q4Rows(pools[0].codes, pools[0].affine.float()), pools[1]), "uint8 codes"),
                       ((k, k, *pools, torch.zeros(3, dtype=torch.int32)), "start is an int32"),
                       ((k, k, *pools, torch.zeros(2)), "start is an int32"),
                       ((k.repeat(1, 3, 1, 1), k.repeat(1, 3, 1, 1), *pools), "9 rows do not fit"),
                       ((k.clone().requires_grad_(), k, *pools), "has no gradient")]:
        with pytest.raises(KernelError, match=words):
            q4.kv_write_paged_q4(*bad)
    assert all(torch.count_nonzero(t) == 0 for pool in pools for t in pool)
    with pytest.raises(KernelError, match="must not be negative"):
        q4.kv_read_paged_q4(*pools, -1)
    with pytest.raises(KernelError, match="start is an int32"):
        q4.kv_read_paged_q4(*pools, 1, torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(KernelError, match="codes \\[B, pages"):
        q4.kv_read_paged_q4(q4.empty_rows(2, channels=64), q4.empty_rows(2, channels=64), 1)


def test_refusals_of_attention_and_linear():
    q, pools, n = torch.zeros(2, 4, 64), _pools(), torch.ones(2, dtype=torch.int32)
    for bad, words in [((q[0], *pools, n), "q is"), ((q.int(), *pools, n), "q is"),
                       ((q[:, :3], *pools, n), "do not share"), ((q[:1], *pools, n), "does not hold 1 sequences"),
                       ((q[..., :32], *_pools(D=128), n), "rows of 32 channels"), ((q, *pools, n[:1]), "lengths is"),
                       ((q, *pools, n.float()), "lengths is"), ((q, *pools, None), "needs the lengths"),
                       ((q, *pools, n, n[:1]), "lo is"), ((q.clone().requires_grad_(), *pools, n), "has no gradient")]:
        with pytest.raises(KernelError, match=words):
            q4.decode_attention_paged_q4(*bad)
    for scale in (float("nan"), float("inf")):
        with pytest.raises(KernelError, match="finite"):
            q4.decode_attention_paged_q4(q, *pools, n, scale=scale)
    w = q4.quantize_rows_q4(torch.randn(5, 70))
    x = torch.zeros(2, 70)
    for bad, words in [((x[:, :64], w), "rows of 64 channels"), ((x.int(), w), "x is"), ((torch.zeros(2, 0), w), "x is"),
                       ((x, q4.quantize_rows_q4(torch.randn(2, 5, 70))), "weights are"),
                       ((x.clone().requires_grad_(), w), "has no gradient")]:
        with pytest.raises(KernelError, match=words):
            q4.linear_q4(*bad)
    with pytest.raises(KernelError, match="floating point"):
        q4.quantize_rows_q4(torch.zeros(3, 4, dtype=torch.int32))
    with torch.no_grad():
        assert q4.linear_q4(x.clone().requires_grad_(), w).shape == (2, 5)
