"""Calls of the 4-bit cache, its weights and its operators at the edges of what they take, on the CPU paths."""

import pytest
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from research_b200.errors import KernelError
from research_b200.infer import quantize_weights
from research_b200.infer.generation import QuantizedKVCache, decode_one, init_kv_cache, prefill
from research_b200.ops import quantized as q4
from tests.test_quantized_generation_cpu import _cache, _model, _rows


# ------------------------------------------------------------------------------------------------- capacity
@pytest.mark.parametrize("bits", [4, 16])
def test_a_step_past_the_cache_is_refused(bits):
    """A cache of 8 rows that is full: no step gets logits that leave its own token out."""

    model = _model()
    cache = init_kv_cache(model, 2, 8, page_size=4, cache_bits=bits)
    prefill(model, torch.randint(0, 256, (2, 7)), cache)
    token = torch.randint(0, 256, (2,))
    assert torch.isfinite(decode_one(model, token, 7, cache)).all()
    for position in (8, 9, 10 ** 6, -1):
        with pytest.raises(IndexError):
            decode_one(model, token, position, cache)
    assert cache.lengths.tolist() == [8, 8]


def test_positions_that_the_cache_does_not_have_are_refused_before_anything_is_written():
    torch.manual_seed(0)
    cache = init_kv_cache(_model(), 2, 8, page_size=4, cache_bits=4)
    H, D = cache.k.codes.shape[2], 16
    tokens = lambda T: (torch.randn(2, T, 2 * H, D), torch.randn(2, T, H, D), torch.randn(2, T, H, D))  # noqa: E731
    cache.update_and_attend(0, *tokens(6), torch.arange(6).expand(2, 6), None)
    held = [t.clone() for pool in (cache.k, cache.v) for t in pool]
    for positions in ([[6, 7, 8, 9, 10]] * 2, [[6, 7, 8], [0, 1, 2]], [[7, 3, 8], [0, 0, 0]], [[-2, -1, 0]] * 2, [[3, -1], [4, 5]],
                      [[8], [0]], [[0], [-1]]):
        at = torch.tensor(positions, dtype=torch.int32)
        with pytest.raises(IndexError, match="8 rows"):
            cache.update_and_attend(0, *tokens(at.shape[1]), at, None)
    assert all(torch.equal(a, b) for a, b in zip(held, [t for pool in (cache.k, cache.v) for t in pool]))
    for positions in ([[6, 7]] * 2, [[7], [7]]):
        at = torch.tensor(positions, dtype=torch.int32)
        assert torch.isfinite(cache.update_and_attend(0, *tokens(at.shape[1]), at, None)).all()


# ------------------------------------------------------------------------------------------------- one prompt for all
@pytest.mark.parametrize("T", [2, 5, 11])
def test_one_prompt_for_every_sequence_of_a_cache(T):
    """As in a 16-bit cache on the GPU: a single prompt goes to all sequences; any other number that is not the cache's is refused."""

    torch.manual_seed(T)
    q, k, v = (torch.randn(1, T, h, 16) for h in (4, 2, 2))
    pos = torch.arange(T, dtype=torch.int32)[None]
    cache, alone = _cache(QuantizedKVCache, batch=3, layers=2), _cache(QuantizedKVCache, batch=1)
    assert torch.equal(cache.update_and_attend(1, q, k, v, pos, None), alone.update_and_attend(0, q, k, v, pos, None))
    for pool, x in ((cache.k, k), (cache.v, v)):
        held = q4.dequantize_rows_q4(q4.quantize_rows_q4(x), 16, torch.float32)
        assert torch.equal(_rows(pool, 1, 3, T, 16), held.expand(3, T, 2, 16))
        assert not pool.codes[0].any() and not pool.affine[0].any()
    before = [t.clone() for pool in (cache.k, cache.v) for t in pool]
    for n, at in ((2, pos), (4, pos), (1, pos + 1), (2, pos[:, :1]), (1, pos[:, :1])):
        t = at.shape[1]
        with pytest.raises(KernelError, match="3 sequences"):
            cache.update_and_attend(1, *(x[:, :t].expand(n, t, *x.shape[2:]) for x in (q, k, v)), at.expand(n, t).contiguous(), None)
    assert all(torch.equal(a, b) for a, b in zip(before, [t for pool in (cache.k, cache.v) for t in pool]))


# ------------------------------------------------------------------------------------------------- channels
def test_rows_of_other_channels_of_the_same_width_are_refused():
    """100 and 120 channels are both stored as 128; rows know which they are."""

    w = q4.quantize_rows_q4(torch.randn(4, 120))
    x = torch.randn(2, 100)
    refused = lambda: pytest.raises(KernelError, match="rows of 100 channels")  # noqa: E731
    with refused():
        q4.linear_q4(x, w)
    with refused():
        q4.linear_q4_reference(x, w)
    with refused():
        q4.dequantize_rows_q4(w, 100)
    assert q4.linear_q4(torch.randn(2, 120), w).shape == (2, 4)
    pools = [q4.empty_rows(2, 3, 2, 4, channels=120) for _ in range(2)]
    right = [q4.empty_rows(2, 3, 2, 4, channels=100) for _ in range(2)]
    rows, n = torch.randn(2, 5, 2, 100), torch.ones(2, dtype=torch.int32)
    for k_pool, v_pool in ((pools[0], pools[1]), (right[0], pools[1]), (pools[0], right[1])):
        with refused():
            q4.kv_write_paged_q4(rows, rows, k_pool, v_pool)
        with refused():
            q4.kv_read_paged_q4(k_pool, v_pool, 1, head_dim=100)
        with refused():
            q4.decode_attention_paged_q4(rows[:, 0], k_pool, v_pool, n)
    assert not any(t.any() for pool in (*pools, *right) for t in pool)
    q4.kv_write_paged_q4(rows, rows, *right)
    back = q4.kv_read_paged_q4(*right, 5, head_dim=100, dtype=torch.float32)[0]
    assert torch.equal(back, q4.dequantize_rows_q4(q4.quantize_rows_q4(rows), 100, torch.float32))
    assert q4.kv_read_paged_q4(*right, 5)[0].shape == (2, 5, 2, 128)                # the stored width, padding and all


def test_rows_keep_their_channels():
    import copy
    import pickle

    w = q4.quantize_rows_q4(torch.randn(4, 120))
    for same in (w, copy.copy(w), copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert type(same) is q4.Q4Rows and same.channels == 120
        assert len(same) == 2 and torch.equal(same.codes, w.codes) and torch.equal(same.affine, w.affine)
    codes, affine = w
    raw = q4.Q4Rows(codes, affine)                                                  # not said: the width alone is looked at
    assert raw.channels is None and q4.Q4Rows(codes, affine, 120).channels == 120
    x = torch.randn(3, 120)
    assert torch.equal(q4.linear_q4(x, raw), q4.linear_q4(x, w))
    cache = _cache(QuantizedKVCache, dim=16)
    assert cache.k.channels == cache._pages(cache.k, 0).channels == 16
    with pytest.raises(KernelError, match="rows of 20 channels"):
        cache.update_and_attend(0, *(torch.randn(2, 1, h, 20) for h in (4, 2, 2)), torch.zeros(2, 1, dtype=torch.int32), None)


# ------------------------------------------------------------------------------------------------- copies of weights
def test_copies_of_weights_may_be_taken_back_in_any_order():
    model = _model()
    p = model.layers[0].attn.wqkv
    owners, rows = [], []
    for _ in range(3):
        owners.append(quantize_weights(model))
        rows.append(p.q4)
    for index, in_use in ((1, 2), (2, 0), (1, 0), (0, None)):           # the latest that is still there; twice is once
        owners[index].remove()
        assert getattr(p, "q4", None) is (None if in_use is None else rows[in_use])
    assert not any(hasattr(p, "q4") for p in model.parameters())
    named = [(p, set(vars(p))) for p in model.parameters()]
    a, b = quantize_weights(model), quantize_weights(model)
    a.remove()
    b.remove()
    assert all(set(vars(p)) == before for p, before in named)           # nothing of it stays


def test_rows_that_a_parameter_had_before_come_back():
    model = _model()
    p = model.layers[0].attn.wo
    p.q4 = mine = q4.quantize_rows_q4(p.detach())
    a = quantize_weights(model)
    with quantize_weights(model):
        a.remove()
        assert p.q4 is not mine
    assert p.q4 is mine
    del p.q4


def test_a_parameter_of_two_modules():
    model = _model()
    model.layers[1].attn.wo = model.layers[0].attn.wo
    p = model.layers[0].attn.wo
    a, b = quantize_weights(model), quantize_weights(model)
    a.remove()
    assert hasattr(p, "q4")
    b.remove()
    assert not hasattr(p, "q4") and not hasattr(p, "q4_copies")


# ------------------------------------------------------------------------------------------------- derivatives
def _calls():
    """Each call with its floating point arguments, by name."""

    w = q4.quantize_rows_q4(torch.randn(5, 70))
    pools = [q4.quantize_rows_q4(torch.randn(2, 2, 2, 4, 64)) for _ in range(2)]
    n = torch.tensor([3, 8])
    held = lambda rows, affine: q4.Q4Rows(rows.codes, affine)  # noqa: E731
    pairs = dict(ka=pools[0].affine, va=pools[1].affine)
    rows = lambda: torch.randn(2, 3, 2, 64)  # noqa: E731
    return [
        (lambda x, a: q4.linear_q4(x, held(w, a)), dict(x=torch.randn(2, 70), a=w.affine)),
        (lambda a: q4.dequantize_rows_q4(held(w, a), 70), dict(a=w.affine)),
        (lambda k, v, ka, va: q4.kv_write_paged_q4(k, v, held(pools[0], ka), held(pools[1], va)), dict(k=rows(), v=rows(), **pairs)),
        (lambda ka, va: q4.kv_read_paged_q4(held(pools[0], ka), held(pools[1], va), 3), pairs),
        (lambda q, ka, va: q4.decode_attention_paged_q4(q, held(pools[0], ka), held(pools[1], va), n),
         dict(q=torch.randn(2, 4, 64), **pairs)),
    ]


@pytest.mark.parametrize("index", range(5))
def test_a_call_that_would_record_a_derivative_is_refused(index):
    call, arguments = _calls()[index]
    call(**arguments)
    for name, value in arguments.items():
        with pytest.raises(KernelError, match="has no gradient"):
            call(**{**arguments, name: value.clone().requires_grad_()})
        with torch.no_grad():
            call(**{**arguments, name: value.clone().requires_grad_()})
            with forward_ad.dual_level():
                with pytest.raises(KernelError, match="no forward-mode derivative"):
                    call(**{**arguments, name: forward_ad.make_dual(value.clone(), torch.ones_like(value))})
                call(**arguments)


def test_quantised_rows_are_plain_data():
    x = torch.randn(3, 70, requires_grad=True)
    rows = q4.quantize_rows_q4(x)
    assert not rows.affine.requires_grad and torch.equal(rows.affine, q4.quantize_rows_q4(x.detach()).affine)
    with forward_ad.dual_level(), pytest.raises(KernelError, match="no forward-mode derivative"):
        q4.quantize_rows_q4(forward_ad.make_dual(x.detach(), torch.ones(3, 70)))


def test_a_linear_with_4_bit_rows_takes_the_parameter_under_a_forward_mode_level():
    from research_b200.ops import functional as Fn

    p = torch.nn.Parameter(torch.randn(5, 70))
    p.q4 = q4.quantize_rows_q4(p)
    x, dx = torch.randn(2, 70), torch.randn(2, 70)
    with torch.no_grad(), forward_ad.dual_level():
        y, dy = forward_ad.unpack_dual(Fn.linear(forward_ad.make_dual(x, dx), p))
        torch.testing.assert_close(y, F.linear(x, p))
        torch.testing.assert_close(dy, F.linear(dx, p))
    with torch.no_grad():
        assert torch.equal(Fn.linear(x, p), q4.linear_q4(x, p.q4))


# ------------------------------------------------------------------------------------------------- kernels that start early
def test_kernels_that_start_early_do_not_take_their_inputs_for_unchanging():
    """What the predecessor may still be writing when a kernel starts is read by plain loads: ``__ldg``, and loads through
    ``const * __restrict__``, are for memory that nothing writes as long as the kernel runs."""

    import re
    from pathlib import Path

    csrc = Path(q4.__file__).parent / "csrc"
    seen = []
    for name in ("quant4.cuh", "quant4.cu", "decode_q4.cu", "linear_q4.cu"):
        text = re.sub(r"//[^\n]*", "", (csrc / name).read_text())
        for head in re.finditer(r"__global__([^{]*?(\w+_kernel)\s*\([^{]*)\{", text):
            depth, at = 1, head.end()
            while depth:
                depth += {"{": 1, "}": -1}.get(text[at], 0)
                at += 1
            body = text[head.end():at]
            if "pdl_wait()" not in body:
                continue
            seen.append(head.group(2))
            assert not re.findall(r"__ldg|ld\.global\.nc|ldcs", body), head.group(2)
            assert not re.findall(r"const\s+[\w:]+\s*\*\s*__restrict__", head.group(1)), head.group(2)
    assert {"kv_write_q4_kernel", "kv_read_q4_kernel", "dequantize_rows_q4_kernel", "decode_q4_kernel", "decode_q4_merge_kernel",
            "linear_q4_few_kernel", "linear_q4_many_kernel", "linear_q4_narrow_kernel"} == set(seen)


# ------------------------------------------------------------------------------------------------- a cache without rows
@pytest.mark.parametrize("pages,page_rows", [(0, 4), (2, 0), (0, 0)])
def test_a_cache_without_rows(pages, page_rows):
    """Rows that the cache does not have are left out, read as zeros, and count for nothing."""

    pools = [q4.empty_rows(2, pages, 2, page_rows, channels=64) for _ in range(2)]
    k = torch.randn(2, 3, 2, 64)
    q4.kv_write_paged_q4(k, k, *pools, torch.tensor([0, 1]))
    for back in q4.kv_read_paged_q4(*pools, 3, torch.tensor([0, 1])):
        assert back.shape == (2, 3, 2, 64) and back.dtype == torch.bfloat16 and not back.any()
    assert not q4.decode_attention_paged_q4(torch.randn(2, 4, 64), *pools, torch.tensor([0, 5])).any()


# ------------------------------------------------------------------------------------------------- shared memory
def test_caches_that_share_memory_are_not_written():
    """K and V rows of one place would be written at once; reading one cache as both is fine."""

    k, v = torch.randn(2, 3, 2, 64), torch.randn(2, 3, 2, 64)
    pool, other = (q4.empty_rows(2, 2, 2, 4, channels=64) for _ in range(2))
    codes, affine = torch.zeros(2 * pool.codes.numel(), dtype=torch.uint8), torch.zeros(2 * pool.affine.numel(), dtype=torch.bfloat16)
    n, m = pool.codes.numel(), pool.affine.numel()
    near = q4.Q4Rows(codes[:n].view(pool.codes.shape), affine[:m].view(pool.affine.shape))
    for same in ((pool, pool), (pool, q4.Q4Rows(pool.codes, other.affine)), (pool, q4.Q4Rows(other.codes, pool.affine)),
                 (near, q4.Q4Rows(codes[32:n + 32].view(pool.codes.shape), affine[m:].view(pool.affine.shape)))):
        with pytest.raises(KernelError, match="share memory"):
            q4.kv_write_paged_q4(k, v, *same)
    assert not any(t.any() for t in (*pool, *other, codes, affine))
    q4.kv_write_paged_q4(k, v, near, q4.Q4Rows(codes[n:].view(pool.codes.shape), affine[m:].view(pool.affine.shape)))
    q4.kv_write_paged_q4(k, v, pool, other)
    assert torch.equal(near.codes, pool.codes) and torch.equal(codes[n:].view(pool.codes.shape), other.codes)
    back = q4.kv_read_paged_q4(pool, pool, 3)
    assert torch.equal(*back)
    q4.decode_attention_paged_q4(torch.randn(2, 4, 64), pool, pool, torch.tensor([1, 3]))


# ------------------------------------------------------------------------------------------------- positions in place
@pytest.mark.parametrize("layer", [0, 1])
def test_positions_that_change_in_place_are_seen_by_every_layer(layer):
    """A program's own position buffer, moved on by fill_ between two steps through a part of the layers."""

    torch.manual_seed(0)
    cache, fresh = (_cache(QuantizedKVCache, layers=2) for _ in range(2))
    at = torch.zeros(2, 1, dtype=torch.int32)
    for position in range(5):
        at.fill_(position)
        q, k, v = (torch.randn(2, 1, h, 16) for h in (4, 2, 2))
        got = cache.update_and_attend(layer, q, k, v, at, 3)
        assert torch.equal(got, fresh.update_and_attend(layer, q, k, v, at.clone(), 3))
    assert all(torch.equal(a, b) for x, y in ((cache.k, fresh.k), (cache.v, fresh.v)) for a, b in zip(x, y))
    with torch.inference_mode():
        got = cache.update_and_attend(0, q, k, v, torch.full((2, 1), 5, dtype=torch.int32), None)
        assert torch.isfinite(got).all()
