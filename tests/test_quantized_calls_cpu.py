"""Calls of the 4-bit cache, its weights and its operators at the edges of what they take, on the CPU paths."""

import pytest
import torch

from research_b200.infer.generation import decode_one, init_kv_cache, prefill
from tests.test_quantized_generation_cpu import _model


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
