"""Calls of the 4-bit cache, its weights and its operators at the edges of what they take, on the CPU paths."""

import pytest
import torch

from research_b200.errors import KernelError
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
