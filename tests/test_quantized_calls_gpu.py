"""Calls of the 4-bit cache, its weights and its operators at the edges of what they take, on the GPU."""

import pytest
import torch

from tests.test_quantized_generation_gpu import _trainer

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


# ------------------------------------------------------------------------------------------------- capacity
@pytest.mark.parametrize("bits", [4, 16])
def test_a_step_past_the_cache_is_refused_on_the_host(bits):
    from research_b200.errors import CacheCapacityError
    from research_b200.infer import decode_one, init_kv_cache, prefill
    from research_b200.infer.generation import GraphedDecodeStep
    from research_b200.ops import native

    model = _trainer().result.model.eval()
    cache = init_kv_cache(model, 2, 16, page_size=8, cache_bits=bits)
    prefill(model, torch.randint(0, 512, (2, 14), device="cuda"), cache)
    token = torch.zeros(2, dtype=torch.int64, device="cuda")
    step = GraphedDecodeStep(model, cache, token, 14)
    held = [t.clone() for pool in (cache.k, cache.v) for t in (pool if bits == 4 else [pool])]
    launches = native.LAUNCHES
    for position in (16, 17, -1):
        for call in (lambda: decode_one(model, token, position, cache), lambda: step(token, position),
                     lambda: GraphedDecodeStep(model, cache, token, position)):
            with pytest.raises(CacheCapacityError):
                call()
    assert native.LAUNCHES == launches
    assert all(torch.equal(a, b) for a, b in zip(held, [t for pool in (cache.k, cache.v) for t in (pool if bits == 4 else [pool])]))
    assert torch.equal(step(token, 15), decode_one(model, token, 15, cache))


def test_a_piece_past_the_cache_is_refused_before_it_is_written():
    from research_b200.errors import CacheCapacityError
    from research_b200.infer import QuantizedKVCache

    cache = QuantizedKVCache(layers=1, batch=2, max_len=8, kv_heads=2, head_dim=64, page_size=4, dtype=BF16,
                             device=torch.device("cuda"))
    held = [t.clone() for pool in (cache.k, cache.v) for t in pool]
    for positions in ([[6, 7, 8, 9]] * 2, [[6, 7, 8], [0, 1, 2]], [[7, 3, 8], [0, 0, 0]], [[-2, -1, 0]] * 2):
        at = torch.tensor(positions, dtype=torch.int32, device="cuda")
        q, k, v = (torch.randn(2, at.shape[1], h, 64, device="cuda", dtype=BF16) for h in (4, 2, 2))
        with pytest.raises(CacheCapacityError):
            cache.update_and_attend(0, q, k, v, at, None)
    assert all(torch.equal(a, b) for a, b in zip(held, [t for pool in (cache.k, cache.v) for t in pool]))


# ------------------------------------------------------------------------------------------------- addresses
def _same(a, b):
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def _off_16(rows, bytes_off):
    """The same 4-bit rows with their pairs ``bytes_off`` bytes behind an address of 16 bytes."""

    from research_b200.ops import quantized as q4

    n = bytes_off // 2
    flat = torch.empty(rows.affine.numel() + 8, dtype=BF16, device="cuda")
    pairs = flat[n:n + rows.affine.numel()].view(rows.affine.shape)
    pairs.copy_(rows.affine)
    assert pairs.data_ptr() % 16 == bytes_off
    return q4.Q4Rows(rows.codes.clone(), pairs)


@pytest.mark.parametrize("D,off", [(64, 4), (64, 8), (64, 12), (128, 8)])
def test_pairs_of_a_cache_start_anywhere_that_a_row_may(D, off):
    """The cache calls read a row's pairs, 4 bytes (heads of 64) or 8 (of 128), at a time."""

    from research_b200.ops import quantized as q4

    g = torch.Generator(device="cuda").manual_seed(D + off)
    B, pages, H, ps, T = 2, 3, 3, 25, 40
    k, v = (torch.randn(B, T, H, D, generator=g, device="cuda").to(BF16) for _ in range(2))
    q = torch.randn(B, 2 * H, D, generator=g, device="cuda").to(BF16)
    plain = [q4.empty_rows(B, pages, H, ps, channels=D, device="cuda") for _ in range(2)]
    odd = [_off_16(pool, off) for pool in plain]
    start = torch.tensor([0, 31], device="cuda", dtype=torch.int32)
    for pools in (plain, odd):
        q4.kv_write_paged_q4(k, v, *pools, start)
    for a, b in zip(plain, odd):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.affine, b.affine)
    for a, b in zip(q4.kv_read_paged_q4(*plain, T, start), q4.kv_read_paged_q4(*odd, T, start)):
        assert torch.equal(a, b)
    assert torch.equal(q4.decode_attention_paged_q4(q, *plain, start + T, start), q4.decode_attention_paged_q4(q, *odd, start + T, start))
    assert torch.equal(q4.dequantize_rows_q4(plain[0], D), q4.dequantize_rows_q4(odd[0], D))


@pytest.mark.parametrize("K,off", [(50, 4), (64, 12), (100, 8), (300, 8), (2048, 8)])
@pytest.mark.parametrize("rows", [1, 12, 40, 90, 2000])
def test_pairs_of_weights_start_anywhere_that_a_row_may(K, off, rows):
    from research_b200.ops import quantized as q4

    g = torch.Generator(device="cuda").manual_seed(K + rows)
    w = q4.quantize_rows_q4(torch.randn(203, K, generator=g, device="cuda"))
    x = torch.randn(rows, K, generator=g, device="cuda").to(BF16)
    want = q4.linear_q4(x, w)
    assert torch.equal(q4.linear_q4(x, _off_16(w, off)), want)
    # weight rows of a larger matrix
    part = q4.Q4Rows(w.codes[1:], w.affine[1:])
    assert torch.equal(q4.linear_q4(x, part), q4.linear_q4(x, q4.Q4Rows(*(t.clone() for t in part))))
    assert _same(q4.dequantize_rows_q4(part, K), q4.dequantize_rows_q4(w, K)[1:])


@pytest.mark.parametrize("D,H,page,pages", [(64, 2, 25, 1), (64, 1, 7, 3), (64, 3, 1, 5), (128, 1, 5, 1)])
def test_layers_of_a_cache_of_odd_pages(D, H, page, pages):
    """Each layer of a cache is a slice; the second one's pairs start where the first one's end."""

    from research_b200.infer import QuantizedKVCache

    caches = [QuantizedKVCache(layers=layers, batch=1, max_len=page * pages, kv_heads=H, head_dim=D, page_size=page,
                               dtype=BF16, device=torch.device("cuda")) for layers in (3, 1)]
    end = min(page * pages, 5)
    for first, T in ((0, end - 1), (end - 1, 1)):
        at = (torch.arange(T, dtype=torch.int32, device="cuda") + first)[None]
        q, k, v = (torch.randn(1, T, h, D, device="cuda", dtype=BF16) for h in (2 * H, H, H))
        want = caches[1].update_and_attend(0, q, k, v, at, None)
        for layer in range(3):
            assert torch.equal(caches[0].update_and_attend(layer, q, k, v, at, None), want)


@pytest.mark.parametrize("D", [64, 128])
def test_dense_keys_values_and_queries_start_on_any_address(D):
    from research_b200.ops import quantized as q4

    B, T, H = 2, 7, 2
    dense = lambda n, *shape: torch.randn(n + 1, device="cuda").to(BF16)[1:].view(shape)  # noqa: E731
    k, v = (dense(B * T * H * D, B, T, H, D) for _ in range(2))
    q = dense(B * 4 * D, B, 4, D)
    assert all(t.is_contiguous() and t.data_ptr() % 16 == 2 for t in (k, v, q))
    pools, same = ([q4.empty_rows(B, 2, H, 5, channels=D, device="cuda") for _ in range(2)] for _ in range(2))
    q4.kv_write_paged_q4(k, v, *pools)
    q4.kv_write_paged_q4(k.clone(), v.clone(), *same)
    assert all(torch.equal(a, b) for x, y in zip(pools, same) for a, b in zip(x, y))
    n = torch.tensor([7, 3], device="cuda")
    assert torch.equal(q4.decode_attention_paged_q4(q, *pools, n), q4.decode_attention_paged_q4(q.clone(), *pools, n))


# ------------------------------------------------------------------------------------------------- one prompt for all
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (torch.float32, 64)])
def test_one_prompt_for_every_sequence_of_a_cache(dtype, D):
    from research_b200.errors import KernelError
    from research_b200.infer import QuantizedKVCache
    from research_b200.ops import quantized as q4

    T = 133
    cache = QuantizedKVCache(layers=2, batch=3, max_len=T + 5, kv_heads=2, head_dim=D, page_size=24, dtype=dtype,
                             device=torch.device("cuda"))
    q, k, v = (torch.randn(1, T, h, D, device="cuda", dtype=dtype) for h in (4, 2, 2))
    pos = torch.arange(T, device="cuda", dtype=torch.int32)[None]
    with cache.prompt():
        got = cache.update_and_attend(1, q, k, v, pos, None)
    alone = QuantizedKVCache(layers=1, batch=1, max_len=T + 5, kv_heads=2, head_dim=D, page_size=24, dtype=dtype,
                             device=torch.device("cuda"))
    assert torch.equal(got, alone.update_and_attend(0, q, k, v, pos, None))
    for pool, x in ((cache.k, k), (cache.v, v)):
        held = q4.quantize_rows_q4(x)
        at = torch.arange(T, device="cuda")
        pages = cache._pages(pool, 1)
        assert torch.equal(pages.codes[:, at // 24, :, at % 24].transpose(0, 1), held.codes.expand(3, -1, -1, -1))
        assert torch.equal(pages.affine[:, at // 24, :, at % 24].transpose(0, 1), held.affine.expand(3, -1, -1, -1, -1))
    for n, at in ((2, pos), (4, pos), (1, pos[:, :9] + 1), (2, pos[:, :1])):
        t = at.shape[1]
        with pytest.raises(KernelError, match="3 sequences"):
            cache.update_and_attend(1, *(x[:, :t].expand(n, t, *x.shape[2:]) for x in (q, k, v)), at.expand(n, t).contiguous(), None)


# ------------------------------------------------------------------------------------------------- derivatives
def test_forward_mode_tangents_are_not_dropped():
    from torch.autograd import forward_ad

    from research_b200.errors import KernelError
    from research_b200.ops import functional as Fn
    from research_b200.ops import quantized as q4

    w = q4.quantize_rows_q4(torch.randn(40, 128, device="cuda"))
    p = torch.nn.Parameter(torch.randn(40, 128, device="cuda"))
    p.q4 = w
    pools = [q4.quantize_rows_q4(torch.randn(2, 2, 2, 8, 64, device="cuda")) for _ in range(2)]
    n = torch.tensor([3, 8], device="cuda")
    with torch.no_grad(), forward_ad.dual_level():
        dual = lambda *shape: forward_ad.make_dual(*(torch.randn(*shape, device="cuda").to(BF16) for _ in range(2)))  # noqa: E731
        row = dual(2, 1, 2, 64)
        for call in (lambda: q4.linear_q4(dual(3, 128), w), lambda: q4.kv_write_paged_q4(row, row, *pools),
                     lambda: q4.decode_attention_paged_q4(dual(2, 4, 64), *pools, n), lambda: q4.quantize_rows_q4(dual(3, 128))):
            with pytest.raises(KernelError, match="no forward-mode derivative"):
                call()
        for rows in (1, 100):                              # the parameter's own kernels have none either, and say so
            with pytest.raises(RuntimeError):
                Fn.linear(dual(rows, 128), p)
    with torch.no_grad():
        x = torch.randn(3, 128, device="cuda").to(BF16)
        assert torch.equal(Fn.linear(x, p), q4.linear_q4(x, w))


# ------------------------------------------------------------------------------------------------- graphs
def test_a_captured_step_keeps_the_copies_of_weights_that_it_reads():
    from research_b200.infer import init_kv_cache, prefill, quantize_weights
    from research_b200.infer.generation import GraphedDecodeStep

    model = _trainer().result.model.eval()
    cache = init_kv_cache(model, 2, 64, cache_bits=4)
    token = torch.tensor([5, 7], device="cuda")
    with quantize_weights(model):
        prefill(model, torch.randint(0, 512, (2, 40), device="cuda"), cache)
        places = {p.q4.codes.data_ptr() for p in model.parameters() if hasattr(p, "q4")}
        sizes = [t.numel() * t.element_size() for p in model.parameters() if hasattr(p, "q4") for t in p.q4]
        step = GraphedDecodeStep(model, cache, token, 40)
        want = step(token, 40).clone()
    assert not any(hasattr(p, "q4") for p in model.parameters())
    other = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(2)]
    assert not places & {t.data_ptr() for t in other}           # the rows are still the step's
    assert torch.equal(step(token, 40), want)


# ------------------------------------------------------------------------------------------------- kernels that start early
@pytest.mark.parametrize("rows", [1, 16, 40, 200])
def test_weights_that_the_predecessor_has_just_written(rows):
    """A cache's rows as weights: each product starts before the write of its weights has ended, and waits for it."""

    from research_b200.ops import quantized as q4

    g = torch.Generator(device="cuda").manual_seed(rows)
    N, D = 4096, 128
    pools = [q4.empty_rows(1, 1, 1, N, channels=D, device="cuda") for _ in range(2)]
    weights = [q4.Q4Rows(*(t.view(N, -1) if i == 0 else t.view(N, 2, 2) for i, t in enumerate(pool)), D) for pool in pools]
    x = torch.randn(rows, D, generator=g, device="cuda").to(BF16)
    full = [torch.randn(2, 1, N, 1, D, generator=g, device="cuda").to(BF16) for _ in range(2)]
    want = [[q4.linear_q4(x, q4.quantize_rows_q4(t.view(N, D))) for t in pair] for pair in full]
    back = [[q4.dequantize_rows_q4(q4.quantize_rows_q4(t.view(N, D)), D) for t in pair] for pair in full]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for pair in full:
            q4.kv_write_paged_q4(*pair, *pools)
            got.append([q4.linear_q4(x, w) for w in weights])
            q4.kv_write_paged_q4(*pair, *pools)
            got[-1].append(q4.dequantize_rows_q4(weights[0], D))
        for a, b, c in zip(got, want, back):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2], c[0])


# ------------------------------------------------------------------------------------------------- precision
@pytest.mark.parametrize("D,G", [(128, 2), (128, 4), (64, 4), (64, 8), (128, 7)])
def test_weights_are_rounded_to_neither_side(D, G):
    """Rows in pairs of one key and opposite values: every weight's share cancels, and what is left is what the weights'
    two bf16 parts lost.

    With s = 1, values of +- 7.5 are the codes 15 and 0 of z = -7.5: a channel is 15 sum p over one row of each pair, less
    7.5 sum p over all.  The low part of a weight is below 2^-7 of it and is rounded by 2^-8 of itself at most, to either
    side: N such errors add up to 15 * 6 * 2^-15 sqrt(sum p^2) but once in 10^7.  A tile's sums are made in fp32 (4 products
    of 2^-22, 14 additions of 2^-24, of 7.5), and its own two sums cancel before tiles are joined.  Cut off instead of
    rounded, the weights would lose 2^-16 each on average, to one side."""

    from research_b200.ops import quantized as q4

    g = torch.Generator(device="cuda").manual_seed(D + G)
    rows, ps = 8192, 128
    k = torch.randn(1, rows // 2, 1, D, generator=g, device="cuda").repeat_interleave(2, 1)
    sign = 1.0 - 2.0 * ((torch.arange(rows, device="cuda")[:, None] + torch.arange(D, device="cuda")) % 2)
    v = (7.5 * sign)[None, :, None]
    pools = [q4.quantize_rows_q4(t.reshape(1, rows // ps, ps, 1, D).transpose(2, 3).contiguous().to(BF16)) for t in (k, v)]
    assert (pools[1].affine[..., 0] == 1.0).all() and (pools[1].affine[..., 1] == -7.5).all()
    q = (0.8 * torch.randn(1, G, D, generator=g, device="cuda")).to(BF16)
    n = torch.tensor([rows], device="cuda", dtype=torch.int32)
    got = q4.decode_attention_paged_q4(q, *pools, n).double().view(G, D)
    keys = q4.dequantize_rows_reference(pools[0], D, torch.float64).transpose(2, 3).reshape(rows, D)
    p = torch.softmax(q[0].double() @ keys.t() * D ** -0.5, -1)
    assert torch.equal(p[:, 0::2], p[:, 1::2])
    tol = 15 * 6 * 2.0 ** -15 * p[:, 0::2].square().sum(-1).sqrt() + 7.5 * (4 * 2.0 ** -22 + 14 * 2.0 ** -24)
    assert (got.abs() <= tol[:, None]).all(), (got.abs().amax(-1) / tol, got.mean(-1))


def bf16_weights_tolerance(x, full):
    """What a product of bf16 ``x`` and ``full`` (float64 copies) with fp32 sums may be off by: half a bf16 step of the result,
    and of the sum's running value, a walk of K products that stays within 5 of its standard deviations, four units of
    2^-24 for each of the K / 16 products that are added to it, and for the joining of up to 8 slices."""

    want = x @ full.t()
    walk = 5 * (x.square() @ full.t().square()).sqrt()
    return want, 2.0 ** -8 * want.abs() + (x.shape[1] / 16 + 8) * 2.0 ** -22 * walk


@pytest.mark.parametrize("rows,N,K", [(17, 2048, 2048), (32, 1000, 1856), (64, 77, 5632), (33, 130, 705), (16, 5000, 4000), (9, 100, 17000),
                                      (1, 100, 33000), (100, 1000, 4000), (128, 9, 16000), (777, 512, 1100), (300, 2600, 520),
                                      (129, 333, 705), (1000, 4096, 300), (65, 1000, 130), (70, 50, 64), (2000, 700, 2048)])
def test_products_of_many_rows_are_those_of_the_weights_as_bf16(rows, N, K):
    """Above few_rows every weight counts as a bf16, one number: against those in 64 bits the result has nothing but its own
    rounding and that of the sums left, which a channel or a bit of a weight more or less is far above."""

    from research_b200.ops import quantized as q4

    assert rows > q4.few_rows(N, K)
    g = torch.Generator(device="cuda").manual_seed(rows + K)
    x = torch.randn(rows, K, generator=g, device="cuda").to(BF16)
    w = q4.quantize_rows_q4(torch.randn(N, K, generator=g, device="cuda") * 0.05)
    want, tol = bf16_weights_tolerance(x.double(), q4.dequantize_rows_reference(w, K, BF16).double())
    off = (q4.linear_q4(x, w).double() - want).abs()
    assert (off <= tol).all(), (off / tol).max()


@pytest.mark.parametrize("kind", ["decoder", "trinity"])
def test_logits_with_4_bit_weights_are_those_of_a_model_that_holds_their_values(kind):
    """A prompt and a step through 4-bit weights, against the same model with the values put in place of its parameters.

    Both multiply the same numbers, but for the step, whose weights are not rounded to bf16; the rest is the bf16 roundings of
    two layers' activations, 2^-8 each, of which two dozen in a row add up to 2^-8 sqrt(24) < 2^-5 of the logits' norm.  What
    4 bits cost themselves is more than that."""

    from research_b200.infer import decode_one, init_kv_cache, prefill, quantize_weights
    from research_b200.ops import quantized as q4

    model = _trainer(kind).result.model.eval()
    g = torch.Generator(device="cuda").manual_seed(1)
    prompts = torch.randint(0, 512, (2, 40), generator=g, device="cuda")
    token = torch.tensor([3, 400], device="cuda")

    @torch.no_grad()
    def logits():
        cache = init_kv_cache(model, 2, 64)
        return [prefill(model, prompts, cache).double(), decode_one(model, token, 40, cache).double()]

    before = logits()
    with quantize_weights(model), torch.no_grad():
        got = logits()
        held = [(p, p.q4) for p in model.parameters() if hasattr(p, "q4")]
    assert len(held) >= 8
    with torch.no_grad():
        for p, rows in held:
            p.copy_(q4.dequantize_rows_q4(rows, p.shape[1]))
            if getattr(p, "shadow", None) is not None:
                p.shadow.copy_(p)
    for a, b, c in zip(got, logits(), before):
        assert (a - b).norm() <= 2.0 ** -5 * b.norm(), (a - b).norm() / b.norm()
        assert (a - c).norm() > 2.0 ** -5 * c.norm(), (a - c).norm() / c.norm()


def test_who_multiplies_is_said_once():
    """The kernel for few rows runs where few_rows says so, and the launcher refuses what it has no room for."""

    from research_b200.ops import native
    from research_b200.ops import quantized as q4

    def launch(rows, K, cluster):
        x = torch.zeros(rows, K, device="cuda", dtype=BF16)
        w = q4.empty_rows(8, channels=K, device="cuda")
        out = torch.empty(rows, 8, device="cuda", dtype=BF16)
        return native.load().b200_q4_linear(x.data_ptr(), K, w.codes.data_ptr(), w.affine.data_ptr(), out.data_ptr(), 8, rows, 8, K,
                                            cluster, native.status_word(x.device).data_ptr(), native._stream())

    for K in (128, 1000, 2048, 2056, 16384, 16392, 32768, 32776):
        rows = q4.few_rows(8, K)
        assert rows in (0, 8, 16) and (rows == 0 or launch(rows, K, 0) == 0)
    for rows, K, cluster in ((17, 128, 0), (9, 16392, 0), (1, 32776, 0), (1, 256, 3), (1, 256, -1), (1, 256, 16)):
        assert launch(rows, K, cluster) == -2
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------- waits that ran out
@pytest.mark.parametrize("bits", [4, 16])
def test_generation_says_when_a_wait_ran_out(bits):
    """A kernel whose bounded wait runs out sets the status word and leaves zeros: no tokens are made of them."""

    from research_b200.errors import KernelError
    from research_b200.infer import generate_tokens
    from research_b200.ops import native

    model = _trainer().result.model.eval()
    prompts = torch.randint(0, 512, (2, 20), device="cuda")
    call = lambda: generate_tokens(model, prompts, max_new_tokens=3, top_k=1, cache_bits=bits, weight_bits=bits)  # noqa: E731
    want = call().generated_ids
    native.status_word(prompts.device)[0:1].fill_(42)
    with pytest.raises(KernelError, match="ran out"):
        call()
    assert call().generated_ids == want and not any(hasattr(p, "q4") for p in model.parameters())


# ------------------------------------------------------------------------------------------------- positions in place
@pytest.mark.parametrize("bits", [4, 16])
def test_positions_that_change_in_place_are_seen_by_every_layer(bits):
    from research_b200.infer import QuantizedKVCache
    from research_b200.infer.generation import PagedKVCache

    kind = QuantizedKVCache if bits == 4 else PagedKVCache
    cache, fresh = (kind(layers=2, batch=2, max_len=128, kv_heads=2, head_dim=64, page_size=64, dtype=BF16,
                         device=torch.device("cuda")) for _ in range(2))
    at = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    for position in range(4):
        at.fill_(position)
        q, k, v = (torch.randn(2, 1, h, 64, device="cuda", dtype=BF16) for h in (4, 2, 2))
        got = cache.update_and_attend(1, q, k, v, at, None)
        assert torch.equal(got, fresh.update_and_attend(1, q, k, v, at.clone(), None))
    pools = [[t for pool in (c.k, c.v) for t in (pool if bits == 4 else [pool])] for c in (cache, fresh)]
    assert all(torch.equal(a, b) for a, b in zip(*pools))
