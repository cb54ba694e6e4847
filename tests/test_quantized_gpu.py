"""4-bit rows on the GPU: codes bit for bit against the restatement, attention and linears against 64 bits.

Tolerances count roundings.  A bf16 result is off by 2^-8 of itself at most (half a step).  In front of that, sums of
products ``x n`` are formed in fp32, in the tensor cores' order: a chain of at most 8 additions per group of 64, each off by
2^-23 of a running sum that is at most ``sum |x| (16 s + |z|)`` in the result's units, hence 2^-20 of that.
"""

import math

import pytest
import torch

from research_b200.errors import KernelError
from research_b200.ops import quantized as q4

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _same(a, b):
    """Bit for bit, NaN equal to NaN."""

    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def _rows_of_all_kinds(g, *shape):
    """Normal rows, some of them constant, shifted, of very wide range, on a coarse grid that makes ties, or without numbers."""

    x = torch.randn(shape, generator=g, device="cuda")
    rows = x.view(-1, shape[-1])
    kind = torch.randint(0, 10, (rows.shape[0],), generator=g, device="cuda")
    rows[kind == 0] = 0.75
    rows[kind == 1] += 100.0
    wide = torch.randint(-60, 20, rows[kind == 2].shape, generator=g, device="cuda")
    rows[kind == 2] *= torch.pow(2.0, wide.float())
    rows[kind == 3] = (rows[kind == 3] * 8).round() / 4
    rows[kind == 4] *= 1e-38
    odd = (kind == 5).nonzero()[:, 0]
    if odd.numel():
        at = torch.randint(0, shape[-1], (odd.numel(),), generator=g, device="cuda")
        rows[odd, at] = torch.tensor([math.nan, math.inf, -math.inf], device="cuda")[odd % 3]
    return x.to(BF16)


# ------------------------------------------------------------------------------------------------- rows
@pytest.mark.parametrize("channels", [1, 5, 63, 64, 65, 128, 129, 200, 777, 2048])
def test_quantize_rows_bit_for_bit(channels):
    g = _gen(channels)
    x = _rows_of_all_kinds(g, 300, channels)
    wider = torch.zeros(300, channels + 3, device="cuda", dtype=BF16)
    wider[:, 1:channels + 1] = x
    want = q4.quantize_rows_reference(x)
    for view in (x, wider[:, 1:channels + 1]):
        got = q4.quantize_rows_q4(view)
        assert torch.equal(got.codes, want.codes) and _same(got.affine, want.affine)
    back = q4.dequantize_rows_q4(got, channels)
    assert _same(back, q4.dequantize_rows_reference(want, channels, BF16))


def test_ties_and_near_ties_bit_for_bit():
    """Every quotient sits on a border or a hair beside one: least -1, step 2, values k + 1/2 steps up, plus 2^-j."""

    n = 4096
    x = torch.zeros(n, 64)
    x[:, 0], x[:, 1] = -1.0, 29.0
    k = torch.arange(n) % 15
    for c in range(2, 64):
        hair = 0.0 if c % 3 == 0 else (1 if c % 3 == 1 else -1) * 2.0 ** -(c % 40)
        base = torch.where(torch.arange(n) % 2 == 0, 0.0, (2.0 * k))
        x[:, c] = base + hair                                            # -1 + (k + 1/2) 2 = 2 k
    x = x.clamp(-1.0, 29.0).to(BF16)
    got, want = q4.quantize_rows_q4(x.cuda()), q4.quantize_rows_q4(x)
    assert torch.equal(got.codes.cpu(), want.codes) and torch.equal(got.affine.cpu(), want.affine)


# ------------------------------------------------------------------------------------------------- cache
@pytest.mark.parametrize("B,T,H,D,pages,ps", [(1, 1, 8, 128, 3, 128), (5, 1, 3, 64, 4, 24), (3, 77, 2, 128, 5, 20),
                                              (2, 300, 4, 64, 3, 128), (2, 129, 1, 128, 200, 1), (4, 33, 8, 64, 2, 100),
                                              (1, 4100, 2, 128, 33, 128)])
def test_write_and_read_bit_for_bit(B, T, H, D, pages, ps):
    g = _gen(B * T + D)
    packed = _rows_of_all_kinds(g, B, T, 3 * H, D).view(B, T, 3 * H * D)            # k and v as columns of a projection
    k, v = (packed[..., i * H * D:(i + 1) * H * D].view(B, T, H, D) for i in (1, 2))
    start = torch.randint(-3, pages * ps, (B,), generator=g, device="cuda", dtype=torch.int32)
    for at in (start, start.long(), None):
        if at is None and T > pages * ps:
            continue
        ours, plain = ([q4.empty_rows(B, pages, H, ps, channels=D, device="cuda") for _ in range(2)] for _ in range(2))
        for pool in ours + plain:
            pool.codes.fill_(9)
            pool.affine.fill_(0.5)
        q4.kv_write_paged_q4(k, v, *ours, at)
        q4.kv_write_paged_q4_reference(k, v, *plain, at)
        for a, b in zip(ours, plain):
            assert torch.equal(a.codes, b.codes) and _same(a.affine, b.affine)
        got = q4.kv_read_paged_q4(*ours, T, at)
        want = q4.kv_read_paged_q4_reference(*plain, T, at, channels=D)
        assert _same(got[0], want[0]) and _same(got[1], want[1])
    assert q4.kv_read_paged_q4(*ours, 0)[0].shape == (B, 0, H, D)


def test_write_takes_rows_of_any_layout():
    g = _gen(0)
    B, T, H, D = 2, 9, 4, 64
    base = torch.randn(B, H, T, D + 4, generator=g, device="cuda").to(BF16)
    k, v = base[..., 1:D + 1].transpose(1, 2), base[..., 3:D + 3].transpose(1, 2)   # heads apart, rows unaligned
    ours, plain = ([q4.empty_rows(B, 2, H, 8, channels=D, device="cuda") for _ in range(2)] for _ in range(2))
    q4.kv_write_paged_q4(k, v, *ours)
    q4.kv_write_paged_q4_reference(k, v, *plain)
    assert all(torch.equal(a, b) for x, y in zip(ours, plain) for a, b in zip(x, y))
    one = k[:1].expand(B, T, H, D)                                                 # one prompt for every sequence
    q4.kv_write_paged_q4(one, one, *ours)
    q4.kv_write_paged_q4_reference(one, one, *plain)
    assert all(torch.equal(a, b) for x, y in zip(ours, plain) for a, b in zip(x, y))


# ------------------------------------------------------------------------------------------------- attention
def _attention64(q, k_pool, v_pool, lengths, lo, scale):
    """Result in 64 bits, and the tolerance of the kernel's (see above): ``2^-8 |o|`` for the result, and for what a score is
    off by, ``d = 2^-20 scale sum |q| (16 s + |z|)``, 2 d of every weight, plus 2^-13 for the weights' own roundings (two
    bf16 parts: 2^-15; exponential, sums, tile-wise rescaling)."""

    B, Hq, D = q.shape
    _, pages, Hkv, ps, _ = k_pool.codes.shape
    G, rows = Hq // Hkv, pages * ps
    dense = [q4.dequantize_rows_reference(p, D, torch.float64).transpose(2, 3).reshape(B, rows, Hkv, D) for p in (k_pool, v_pool)]
    most = [(p.affine[..., 0].double().abs() * m + p.affine[..., 1].double().abs()).repeat_interleave(64, -1)
            .transpose(2, 3).reshape(B, rows, Hkv, D) for p, m in ((k_pool, 16), (v_pool, 15))]
    out, tol = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda"), torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        first = 0 if lo is None else max(int(lo[b]), 0)
        last = min(int(lengths[b]), rows)
        if first >= last:
            continue
        k, v, km, vm = (t[b, first:last].repeat_interleave(G, 1) for t in (*dense, *most))
        qd = q[b].double()
        p = torch.softmax(torch.einsum("hd,rhd->hr", qd, k) * scale, -1)
        d = 2.0 ** -20 * abs(scale) * torch.einsum("hd,rhd->hr", qd.abs(), km)
        out[b] = torch.einsum("hr,rhd->hd", p, v)
        tol[b] = 2.0 ** -8 * out[b].abs() + torch.einsum("hr,rhd->hd", p * (2 * d.amax(-1, keepdim=True) + 2.0 ** -13), vm)
    return out.view(B, -1), tol.view(B, -1)


def _pools(g, B, pages, H, ps, D, spread=1.0):
    return [q4.quantize_rows_reference((torch.randn(B, pages, H, ps, D, generator=g, device="cuda") * spread
                                        + 0.4 * torch.randn(D, generator=g, device="cuda")).to(BF16)) for _ in range(2)]


@pytest.mark.parametrize("D,Hq,Hkv,pages,ps", [
    (128, 16, 8, 9, 128), (128, 8, 8, 20, 64), (64, 12, 4, 50, 24), (64, 8, 1, 11, 100), (128, 8, 1, 300, 4), (128, 5, 1, 8, 128),
    (64, 14, 2, 17, 64), (64, 3, 3, 1200, 1), (128, 32, 8, 5, 256), (128, 6, 1, 70, 16), (64, 4, 1, 3, 512)])
def test_attention_against_64_bits(D, Hq, Hkv, pages, ps):
    g = _gen(D + Hq + ps)
    cap = pages * ps
    lengths = torch.tensor([1, 2, 15, 16, 17, 63, 64, 65, 100, 130, cap - 1, cap, 2 * cap, 0, -5, 500], device="cuda", dtype=torch.int32)
    lo = torch.tensor([0, 1, 14, 16, -9, 62, 0, 64, 37, 129, cap - 300, 5, cap - 1, 0, 0, 499], device="cuda", dtype=torch.int32)
    B = lengths.numel()
    q = torch.randn(B, Hq, D, generator=g, device="cuda").to(BF16)
    k, v = _pools(g, B, pages, Hkv, ps, D)
    for bounds in (None, lo):
        want, tol = _attention64(q, k, v, lengths, bounds, D ** -0.5)
        got = q4.decode_attention_paged_q4(q, k, v, lengths, bounds)
        assert got.dtype == BF16 and got.shape == (B, Hq * D)
        off = (got.double() - want).abs()
        assert (off <= tol).all(), ((off - tol).max(), off.max())
        assert torch.equal(got, q4.decode_attention_paged_q4(q, k, v, lengths, bounds))          # the same bits again
    packed = torch.zeros(B, (Hq + Hkv) * D, device="cuda", dtype=BF16)
    packed[:, :Hq * D] = q.view(B, Hq * D)
    strided = packed[:, :Hq * D].view(B, Hq, D)
    assert torch.equal(q4.decode_attention_paged_q4(strided, k, v, lengths.long(), bounds.long()), got)


@pytest.mark.parametrize("scale", [0.3, -0.1, 0.0])
def test_attention_scales_and_long_rows(scale):
    g = _gen(7)
    B, pages, H, ps, D = 2, 90, 2, 128, 128
    q = torch.randn(B, 4, D, generator=g, device="cuda").to(BF16)
    k, v = _pools(g, B, pages, H, ps, D, 0.5)
    lengths = torch.tensor([pages * ps, 9999], device="cuda", dtype=torch.int32)
    want, tol = _attention64(q, k, v, lengths, None, scale)
    got = q4.decode_attention_paged_q4(q, k, v, lengths, scale=scale)
    off = (got.double() - want).abs()
    assert (off <= tol).all(), (off - tol).max()


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 16, 8), (64, 8, 1), (128, 3, 1)])
def test_masked_rows_may_hold_anything(D, Hq, Hkv):
    g = _gen(D)
    B, pages, ps = 4, 7, 40
    q = torch.randn(B, Hq, D, generator=g, device="cuda").to(BF16)
    k, v = _pools(g, B, pages, Hkv, ps, D)
    lengths = torch.tensor([201, 33, 64, 0], device="cuda", dtype=torch.int32)
    lo = torch.tensor([70, 1, 63, 0], device="cuda", dtype=torch.int32)
    want = q4.decode_attention_paged_q4(q, k, v, lengths, lo)
    at = torch.arange(pages * ps, device="cuda").view(pages, 1, ps)
    for fill in (math.nan, math.inf, -math.inf, 3e38):
        for pool in (k, v):
            for b in range(B):
                hidden = ((at < lo[b]) | (at >= lengths[b])).expand(pages, Hkv, ps)
                pool.affine[b][hidden] = fill
                pool.codes[b][hidden] = 255
        assert torch.equal(q4.decode_attention_paged_q4(q, k, v, lengths, lo), want)
    assert torch.count_nonzero(want[3]) == 0


def test_a_visible_row_without_numbers_shows():
    g = _gen(1)
    q = torch.randn(2, 4, 64, generator=g, device="cuda").to(BF16)
    k, v = _pools(g, 2, 2, 2, 32, 64)
    lengths = torch.tensor([50, 50], device="cuda", dtype=torch.int32)
    clean = q4.decode_attention_paged_q4(q, k, v, lengths).view(2, 2, 2, 64)
    k.affine[0, 1, 0, 3] = math.nan
    v.affine[1, 0, 1, 7] = math.nan
    got = q4.decode_attention_paged_q4(q, k, v, lengths).view(2, 2, 2, 64)
    assert got[0, 0].isnan().all() and got[1, 1].isnan().all()
    assert torch.equal(got[0, 1], clean[0, 1]) and torch.equal(got[1, 0], clean[1, 0])


def test_rows_of_very_different_size():
    """A row of tiny values with nearly all the weight beside rows of huge values with nearly none."""

    g = _gen(5)
    D, pages, ps = 128, 2, 64
    k_rows = torch.randn(1, pages, 1, ps, D, generator=g, device="cuda") * 0.01
    v_rows = torch.randn(1, pages, 1, ps, D, generator=g, device="cuda") * 1e4
    q = torch.ones(1, 2, D, device="cuda", dtype=BF16)
    k_rows[0, 0, 0, 5] = 12.0
    v_rows[0, 0, 0, 5] = torch.randn(D, generator=g, device="cuda") * 1e-6
    k, v = (q4.quantize_rows_reference(t.to(BF16)) for t in (k_rows, v_rows))
    lengths = torch.tensor([100], device="cuda", dtype=torch.int32)
    want, tol = _attention64(q, k, v, lengths, None, D ** -0.5)
    got = q4.decode_attention_paged_q4(q, k, v, lengths)
    assert (want.abs().max() < 1e-5) and ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("D,G", [(128, 4), (64, 8)])
@pytest.mark.parametrize("q_size,k_size,scale", [(5e37, 1e-37, 0.09), (1e-37, 1e37, 0.1), (1.0, 1.0, 0.0), (5e37, 1.0, 0.0),
                                                 (1e-37, 1.0, 1e-38), (3e30, 1e-4, -1e-27), (1.0, 1e35, 1e-36)])
def test_attention_of_extreme_numbers(D, G, q_size, k_size, scale):
    g = _gen(D)
    pages, ps = 3, 40
    q = (torch.randn(3, G, D, generator=g, device="cuda") * q_size).to(BF16)
    q[:, 1] = 0.0
    q[:, 2, D // 2:] = 0.0
    k = q4.quantize_rows_reference((torch.randn(3, pages, 1, ps, D, generator=g, device="cuda") * k_size).to(BF16))
    v_rows = torch.randn(3, pages, 1, ps, D, generator=g, device="cuda")
    v_rows[0] *= 1e37
    v_rows[1, :, :, ::7] *= 1e-30
    v = q4.quantize_rows_reference(v_rows.to(BF16))
    lengths = torch.tensor([70, 120, 1], device="cuda", dtype=torch.int32)
    lo = torch.tensor([66, 0, 0], device="cuda", dtype=torch.int32)
    want, tol = _attention64(q, k, v, lengths, lo, scale)
    off = (q4.decode_attention_paged_q4(q, k, v, lengths, lo, scale).double() - want).abs()
    assert (off <= tol).all(), (off - tol).max()


def test_offsets_past_32_bits():
    """Two caches whose words number more than 2^31."""

    B, D, ps = 2, 128, 128
    pages = 72 * 2 ** 20 // ps
    k, v = (q4.empty_rows(B, pages, 1, ps, channels=D, device="cuda") for _ in range(2))
    assert k.codes.numel() // 4 > 2 ** 31
    g = _gen(2)
    rows = [torch.randn(B, 3, 1, D, generator=g, device="cuda").to(BF16) for _ in range(2)]
    start = torch.tensor([pages * ps - 3, pages * ps - 70], device="cuda", dtype=torch.int32)
    q4.kv_write_paged_q4(*rows, k, v, start)
    back = q4.kv_read_paged_q4(k, v, 3, start)
    small = [q4.quantize_rows_reference(x.transpose(1, 2)[:, None].contiguous()) for x in rows]
    for b, s in zip(back, small):
        assert torch.equal(b, q4.dequantize_rows_reference(s, D, BF16)[:, 0].transpose(1, 2))
    q = torch.randn(B, 4, D, generator=g, device="cuda").to(BF16)
    got = q4.decode_attention_paged_q4(q, k, v, start + 3, start)
    want, tol = _attention64(q, *small, torch.full((B,), 3, device="cuda"), None, D ** -0.5)
    assert ((got.double() - want).abs() <= tol).all()
    del k, v
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------- linear
def _linear64(x, w, K):
    """Result in 64 bits, what the tolerance of codes as they are adds to its rounding, and ``|x| |W|^T``."""

    a, width = w.affine.double(), w.codes.shape[1] * 2
    s, z = a[..., 0].abs(), a[..., 1].abs()
    xd = torch.nn.functional.pad(x.double().abs(), (0, width - K)).unflatten(-1, (-1, 64))          # rows, groups, 64
    full = q4.dequantize_rows_reference(w, K, torch.float64)
    want = x.double() @ full.t()
    sums = xd.sum(-1) @ (16 * s + z).t()                    # 2^-20 per group, and 2^-23 for each of K / 64 additions of groups
    return want, sums * (2.0 ** -20 + 2.0 ** -23 * (K / 64)), x.double().abs() @ full.abs().t()


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 31, 33, 48, 64, 65, 200])
@pytest.mark.parametrize("N,K", [(1, 1), (8, 64), (130, 128), (2048, 2048), (1000, 1856), (333, 705), (77, 5632), (17, 191), (40, 66)])
def test_linear_against_64_bits(rows, N, K):
    g = _gen(rows * 1000 + N)
    x = torch.randn(rows, K, generator=g, device="cuda").to(BF16)
    w = q4.quantize_rows_q4(torch.randn(N, K, generator=g, device="cuda") * 0.05)
    want, sums, plain = _linear64(x, w, K)
    # above few_rows the weights are rounded to bf16 and the sums run over K in one accumulator: to the result's rounding come
    # 2^-8 of each |x w|, and 2^-23 of the running sum for each of K additions
    tol = 2.0 ** -8 * want.abs() + sums
    if rows > q4.few_rows(N, K):
        tol = 2.0 ** -8 * want.abs() + plain * (1.01 * 2.0 ** -8 + 2.0 ** -23 * K)
    got = q4.linear_q4(x, w)
    assert got.shape == (rows, N) and got.dtype == BF16
    off = (got.double() - want).abs()
    assert (off <= tol).all(), ((off - tol).max(), off.max())
    assert torch.equal(got, q4.linear_q4(x, w))
    wider = torch.zeros(rows, K + 5, device="cuda", dtype=BF16)
    wider[:, 3:K + 3] = x
    assert torch.equal(q4.linear_q4(wider[:, 3:K + 3], w), got)                     # rows on odd addresses


@pytest.mark.parametrize("rows,N,K,slices", [(777, 512, 1100, 4), (129, 333, 705, 2), (100, 1000, 4000, 8), (65, 1000, 130, 0),
                                             (1000, 4096, 300, 0), (70, 50, 64, 0), (300, 2600, 520, 2), (128, 9, 16000, 8), (150, 9001, 1000, 1)])
def test_linear_of_many_rows(rows, N, K, slices):
    """Products on tiles of 128 x 128, in each cut of K, and with the weights expanded first."""

    assert q4.linear_slices(rows, N, K) == slices
    g = _gen(rows + K)
    x = torch.randn(rows, K, generator=g, device="cuda").to(BF16)
    x[rows - 1] *= 1e30
    x[0, 5], x[1, 6] = math.nan, math.inf
    w = q4.quantize_rows_q4(torch.randn(N, K, generator=g, device="cuda") * 0.05)
    w.affine[N - 2, 0] = math.nan
    got = q4.linear_q4(x, w)
    assert torch.equal(got[2:, :N - 2], q4.linear_q4(x, w)[2:, :N - 2])                 # the same bits again
    assert got[0].isnan().all() and not got[1].isfinite().any() and got[:, N - 2].isnan().all()
    w.affine[N - 2, 0] = 0.0
    want, _, plain = _linear64(x[2:], w, K)
    off = (got[2:].double() - want).abs()
    off[:, N - 2] = 0.0
    tol = 2.0 ** -8 * want.abs() + plain * (1.01 * 2.0 ** -8 + 2.0 ** -23 * K)
    assert (off <= tol).all(), (off - tol).max()


@pytest.mark.parametrize("rows,N,K", [(1, 20003, 5632), (16, 7200, 2300), (7, 300, 16000), (8, 40, 32768), (11, 100, 16384),
                                      (9, 100, 17000), (1, 100, 33000), (5, 70000, 130), (13, 3001, 999), (2, 17, 4096)])
def test_linear_of_long_rows_and_many_weights(rows, N, K):
    """One block to a row, clusters of two to eight, more tiles than a cluster's blocks hold sums of, and rows too long."""

    g = _gen(rows + K)
    x = torch.randn(rows, K, generator=g, device="cuda").to(BF16)
    w = q4.quantize_rows_q4(torch.randn(N, K, generator=g, device="cuda") * 0.05)
    want, tol, plain = _linear64(x, w, K)
    if rows > q4.few_rows(N, K):
        tol = plain * (1.01 * 2.0 ** -8 + 2.0 ** -23 * K)
    got = q4.linear_q4(x, w)
    off = (got.double() - want).abs()
    assert (off <= 2.0 ** -8 * want.abs() + tol).all(), (off - 2.0 ** -8 * want.abs() - tol).max()
    assert torch.equal(got, q4.linear_q4(x, w))


@pytest.mark.parametrize("rows", [3, 9, 16])
def test_linear_rows_of_uneven_size(rows):
    """A channel of 2^12 times the others' size, a row of tiny values, a row of zeros, one of huge values."""

    g = _gen(rows)
    N, K = 260, 1100
    x = torch.randn(rows, K, generator=g, device="cuda")
    x[0, 77] = 5000.0
    x[1] *= 1e-30
    x[2] = 0.0
    if rows > 3:
        x[rows - 1] *= 1e25
        x[rows - 2] *= torch.pow(2.0, torch.randint(-40, 1, (K,), generator=g, device="cuda").float())
    x = x.to(BF16)
    w = q4.quantize_rows_q4(torch.randn(N, K, generator=g, device="cuda") * 0.05)
    want, tol, _ = _linear64(x, w, K)
    off = (q4.linear_q4(x, w).double() - want).abs()
    assert (off <= 2.0 ** -8 * want.abs() + tol).all(), (off - 2.0 ** -8 * want.abs() - tol).max()
    assert torch.count_nonzero(q4.linear_q4(x, w)[2]) == 0


def test_linear_shapes_and_broadcast_rows():
    g = _gen(0)
    w = q4.quantize_rows_q4(torch.randn(96, 192, generator=g, device="cuda"))
    x = torch.randn(2, 3, 192, generator=g, device="cuda").to(BF16)
    y = q4.linear_q4(x, w)
    assert y.shape == (2, 3, 96) and torch.equal(y.view(6, 96), q4.linear_q4(x.view(6, 192), w))
    assert q4.linear_q4(x[:0], w).shape == (0, 3, 96)
    for rows in (5, 100):
        same = q4.linear_q4(x[0, :1].expand(rows, 192), w)
        assert torch.equal(same, q4.linear_q4(x[0, :1].expand(rows, 192).contiguous(), w))
    assert q4.linear_q4(x.transpose(0, 1), w).shape == (3, 2, 96)
    assert torch.equal(q4.linear_q4(x.transpose(0, 1), w), y.transpose(0, 1))


def test_a_row_of_x_without_numbers_stays_in_its_row():
    g = _gen(3)
    w = q4.quantize_rows_q4(torch.randn(50, 320, generator=g, device="cuda"))
    x = torch.randn(5, 320, generator=g, device="cuda").to(BF16)
    clean = q4.linear_q4(x, w)
    x[2, 7], x[3, 100] = math.nan, math.inf
    got = q4.linear_q4(x, w)
    assert got[2].isnan().all() and not got[3].isfinite().any()
    assert torch.equal(got[[0, 1, 4]], clean[[0, 1, 4]])


# ------------------------------------------------------------------------------------------------- together
def _step(x, q, wk, wo, pools, position):
    """A layer's decode step: projections of the new token, its row into the cache, attention, output projection."""

    B, D = x.shape[0], q.shape[2]
    kv = q4.linear_q4(x, wk).view(B, 1, -1, D)
    H = kv.shape[2] // 2
    q4.kv_write_paged_q4(kv[:, :, :H], kv[:, :, H:], *pools, position)
    return q4.linear_q4(q4.decode_attention_paged_q4(q, *pools, position + 1), wo)


def _step_inputs(seed):
    g = _gen(seed)
    B, H, Hq, D, hidden = 6, 2, 8, 128, 512
    x = torch.randn(B, hidden, generator=g, device="cuda").to(BF16)
    q = torch.randn(B, Hq, D, generator=g, device="cuda").to(BF16)
    wk = q4.quantize_rows_q4(torch.randn(2 * H * D, hidden, generator=g, device="cuda") * 0.05)
    wo = q4.quantize_rows_q4(torch.randn(hidden, Hq * D, generator=g, device="cuda") * 0.05)
    pools = _pools(g, B, 12, H, 64, D)
    position = torch.tensor([0, 5, 63, 64, 400, 767], device="cuda", dtype=torch.int32)
    return x, q, wk, wo, pools, position


def test_a_step_of_all_of_them_and_its_graph():
    x, q, wk, wo, pools, position = _step_inputs(11)
    got = _step(x, q, wk, wo, pools, position)
    kv = q4.linear_q4(x, wk).view(6, 1, 4, 128)
    plain = [q4.Q4Rows(*(t.clone() for t in pool)) for pool in _step_inputs(11)[4]]
    q4.kv_write_paged_q4_reference(kv[:, :, :2], kv[:, :, 2:], *plain, position)
    assert all(torch.equal(a, b) for u, w in zip(pools, plain) for a, b in zip(u, w))
    want, tol = _attention64(q, *plain, position + 1, None, 128 ** -0.5)
    o = q4.decode_attention_paged_q4(q, *pools, position + 1)
    assert ((o.double() - want).abs() <= tol).all()
    y, sums, _ = _linear64(o, wo, 1024)
    assert ((got.double() - y).abs() <= 2.0 ** -8 * y.abs() + sums).all()

    # two graphs of the same step on caches of their own, replayed at the same time on two streams with new inputs
    sides, graphs = [], []
    for seed in (11, 12):
        state = _step_inputs(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(*state)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(*state)
        sides.append(side)
        graphs.append((graph, state, out))
    for seed in (21, 22):
        fresh = [_step_inputs(seed + 100 * i) for i in range(2)]
        for (_, state, _), new in zip(graphs, fresh):
            for old, now in zip((*state[:4], *state[4], state[5]), (*new[:4], *new[4], new[5])):
                for a, b in zip(old, now) if isinstance(old, tuple) else ((old, now),):
                    a.copy_(b)
        torch.cuda.synchronize()
        for _ in range(3):
            for side, (graph, _, _) in zip(sides, graphs):
                with torch.cuda.stream(side):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), new in zip(graphs, fresh):
            assert torch.equal(out, _step(*new))


def test_calls_follow_the_current_stream():
    x, q, wk, wo, pools, position = _step_inputs(3)
    want = _step(x, q, wk, wo, [q4.Q4Rows(*(t.clone() for t in p)) for p in pools], position)
    side = torch.cuda.Stream()
    late = torch.empty_like(x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
        got = _step(late, q, wk, wo, pools, position)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals_on_the_device():
    q = torch.zeros(1, 9, 64, device="cuda", dtype=BF16)
    n = torch.ones(1, device="cuda", dtype=torch.int32)
    pools = [q4.empty_rows(1, 1, 1, 64, channels=64, device="cuda") for _ in range(2)]
    with pytest.raises(KernelError, match="up to 8 query heads"):
        q4.decode_attention_paged_q4(q, *pools, n)
    with pytest.raises(KernelError, match="bf16 queries"):
        q4.decode_attention_paged_q4(q[:, :1].float(), *pools, n)
    with pytest.raises(KernelError, match="all tensors have to be on"):
        q4.decode_attention_paged_q4(q[:, :1], *pools, n.cpu())
    narrow = [q4.empty_rows(1, 1, 1, 64, channels=32, device="cuda") for _ in range(2)]
    with pytest.raises(KernelError, match="head_dim 64 and 128"):
        q4.decode_attention_paged_q4(q[:, :1, :32], *narrow, n)
    rows = torch.zeros(1, 1, 1, 32, device="cuda", dtype=BF16)
    with pytest.raises(KernelError, match="head_dim 64 and 128"):
        q4.kv_write_paged_q4(rows, rows, *narrow)
    with pytest.raises(KernelError, match="bf16 rows"):
        q4.kv_write_paged_q4(q[:, None, :1].float(), q[:, None, :1].float(), *pools)
    w = q4.quantize_rows_q4(torch.zeros(4, 64, device="cuda"))
    with pytest.raises(KernelError, match="takes bf16"):
        q4.linear_q4(torch.zeros(1, 64, device="cuda"), w)
    with pytest.raises(KernelError, match="all tensors have to be on"):
        q4.linear_q4(torch.zeros(1, 64, dtype=BF16), w)
