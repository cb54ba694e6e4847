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
