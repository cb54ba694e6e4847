"""Generation with a 4-bit cache and 4-bit weights on the CPU paths."""

import json
import math
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F

from research_b200.config import run_spec_from_mapping
from research_b200.errors import ContractError, KernelError
from research_b200.infer import QuantizedKVCache, quantize_weights
from research_b200.infer.generation import PagedKVCache, decode_one, generate_tokens, init_kv_cache, prefill
from research_b200.models.build import build_model
from research_b200.ops import quantized as q4
from tests.helpers import tiny_dataset, tiny_raw_config, write_toml


def _model(kind="decoder"):
    spec = run_spec_from_mapping(tiny_raw_config(Path("m.json"), kind=kind))
    return build_model(spec.model, seed=0).model.eval()


def _cache(kind, batch=2, max_len=20, page=4, heads=2, dim=16, layers=1):
    return kind(layers=layers, batch=batch, max_len=max_len, kv_heads=heads, head_dim=dim, page_size=page,
                dtype=torch.float32, device=torch.device("cpu"))


def _rows(pool, layer, B, end, D):
    pages = q4.Q4Rows(*(t[layer].view(B, -1, *t.shape[2:]) for t in pool))
    dense = q4.dequantize_rows_q4(pages, D, torch.float32)
    return dense.permute(0, 1, 3, 2, 4).flatten(1, 2)[:, :end]


def _plain(q, k, v, positions, window):
    B, T, Hq, D = q.shape
    g = Hq // k.shape[2]
    out = torch.zeros(B, T, Hq, D)
    for b in range(B):
        for t in range(T):
            p = int(positions[b, t])
            lo = 0 if window is None else max(p - window + 1, 0)
            for h in range(Hq):
                w = torch.softmax(k[b, lo:p + 1, h // g] @ q[b, t, h] / math.sqrt(D), 0)
                out[b, t, h] = w @ v[b, lo:p + 1, h // g]
    return out.reshape(B, T, Hq * D)


def test_cache_holds_36_bytes_for_64_channels():
    c = _cache(QuantizedKVCache, dim=128, page=8)
    assert c.k.codes.shape == (1, 6, 2, 8, 64) and c.k.affine.shape == (1, 6, 2, 8, 2, 2)
    assert c.page_table.tolist() == [[0, 1, 2], [3, 4, 5]] and c.max_len == 24
    full = _cache(PagedKVCache, dim=128, page=8)
    held = sum(t.numel() * t.element_size() for t in c.k)
    assert held * 128 == full.k.numel() * 2 * 36


@pytest.mark.parametrize("window", [None, 5])
def test_cache_attends_over_what_it_holds(window):
    """A prompt attends over its own rows; steps, later pieces and scattered tokens over the quantised ones."""

    torch.manual_seed(0)
    B, Hq, H, D = 2, 4, 2, 16
    c = _cache(QuantizedKVCache)

    def tokens(T):
        return torch.randn(B, T, Hq, D), torch.randn(B, T, H, D), torch.randn(B, T, H, D)

    at = lambda first, T: (torch.arange(T, dtype=torch.int32) + first).expand(B, T).contiguous()  # noqa: E731
    q, k, v = tokens(6)
    torch.testing.assert_close(c.update_and_attend(0, q, k, v, at(0, 6), window), _plain(q, k, v, at(0, 6), window),
                               atol=1e-5, rtol=0)
    held = [q4.dequantize_rows_q4(q4.quantize_rows_q4(t), D, torch.float32) for t in (k, v)]
    for got, want in zip((c.k, c.v), held):
        assert torch.equal(_rows(got, 0, B, 6, D), want)
    for positions in (at(6, 1), torch.tensor([[7], [3]], dtype=torch.int32), at(8, 4), torch.tensor([[12, 13], [2, 3]], dtype=torch.int32),
                      torch.tensor([[14, 2, 14], [9, 5, 4]], dtype=torch.int32)):
        T = positions.shape[1]
        q, k, v = tokens(T)
        out = c.update_and_attend(0, q, k, v, positions, window)
        end = int(positions.max()) + 1
        kk, vv = _rows(c.k, 0, B, end, D), _rows(c.v, 0, B, end, D)
        new = q4.dequantize_rows_q4(q4.quantize_rows_q4(k), D, torch.float32)
        for b in range(B):
            last = {int(p): t for t, p in enumerate(positions[b])}
            for p, t in last.items():
                assert torch.equal(kk[b, p], new[b, t])
        torch.testing.assert_close(out, _plain(q, kk, vv, positions, window), atol=1e-5, rtol=0)


@pytest.mark.parametrize("kind", ["decoder", "trinity"])
def test_prefill_and_steps_through_a_model(kind):
    """The logits of a step are those of a full-precision cache that was given the quantised rows."""

    torch.manual_seed(1)
    model = _model(kind)
    prompt = torch.randint(0, 256, (2, 7))
    cache = init_kv_cache(model, 2, 16, page_size=4, cache_bits=4)
    assert isinstance(cache, QuantizedKVCache)
    full = init_kv_cache(model, 2, 16, page_size=4)
    assert torch.equal(prefill(model, prompt, cache), prefill(model, prompt, full))
    D = model.spec.head_dim
    for step in range(3):
        for pool, held in ((full.k, cache.k), (full.v, cache.v)):
            pool.copy_(q4.dequantize_rows_q4(held, D, torch.float32))
        token = torch.randint(0, 256, (2,))

        class Rounded(PagedKVCache):
            def update_and_attend(self, layer, q, k, v, positions, window):
                k, v = (q4.dequantize_rows_q4(q4.quantize_rows_q4(t), D, torch.float32) for t in (k, v))
                return super().update_and_attend(layer, q, k, v, positions, window)

        full.__class__ = Rounded
        got, want = decode_one(model, token, 7 + step, cache), decode_one(model, token, 7 + step, full)
        torch.testing.assert_close(got, want, atol=1e-4, rtol=0)
        full.__class__ = PagedKVCache
    assert cache.lengths.tolist() == [10, 10]


def test_generate_with_both_and_refusals():
    model = _model()
    prompt = torch.tensor([[3, 1, 4, 1, 5], [9, 2, 6, 5, 3]])
    plain = generate_tokens(model, prompt, max_new_tokens=4, top_k=1, page_size=4)
    for bits in ((4, 16), (16, 4), (4, 4)):
        out = generate_tokens(model, prompt, max_new_tokens=4, top_k=1, page_size=4, cache_bits=bits[0], weight_bits=bits[1])
        assert [len(g) for g in out.generated_ids] == [4, 4] and all(math.isfinite(x) for r in out.logprobs for x in r)
        again = generate_tokens(model, prompt, max_new_tokens=4, top_k=1, page_size=4, cache_bits=bits[0], weight_bits=bits[1])
        assert out.generated_ids == again.generated_ids
    assert generate_tokens(model, prompt, max_new_tokens=4, top_k=1, page_size=4).generated_ids == plain.generated_ids
    assert not any(hasattr(p, "q4") for p in model.parameters())
    with pytest.raises(ContractError, match="cache_bits must be 4 or 16"):
        generate_tokens(model, prompt, max_new_tokens=1, cache_bits=8)
    with pytest.raises(ContractError, match="weight_bits must be 4 or 16"):
        generate_tokens(model, prompt, max_new_tokens=1, weight_bits=8)
    with pytest.raises(ContractError, match="must be positive"):
        generate_tokens(model, prompt, max_new_tokens=0, weight_bits=4)
    assert not any(hasattr(p, "q4") for p in model.parameters())


@pytest.mark.parametrize("kind", ["decoder", "trinity"])
def test_quantized_weights_are_used_without_gradients_only(kind):
    from research_b200.ops import functional as Fn

    model = _model(kind)
    ids = torch.randint(0, 256, (2, 8))
    with torch.no_grad():
        before = model(ids).logits
    with quantize_weights(model) as held:
        named = {n: p for n, p in model.named_parameters() if hasattr(p, "q4")}
        assert {n.rsplit(".", 1)[1] for n in named} <= {"wqkv", "wo", "wgate", "w_gate_up", "w_down"}
        assert not any(x in n for n in named for x in ("embed", "lm_head", "router", ".experts."))
        assert len(named) >= 4 * model.spec.num_layers - 2
        p = model.layers[0].attn.wqkv
        x = torch.randn(3, p.shape[1])
        with torch.no_grad():
            want = F.linear(x, q4.dequantize_rows_q4(p.q4, p.shape[1], torch.float32))
            assert torch.equal(Fn.linear(x, p), want) and not torch.equal(Fn.linear(x, p), F.linear(x, p))
            assert not torch.equal(model(ids).logits, before)
        x.requires_grad_()
        y = Fn.linear(x, p)
        assert torch.equal(y, F.linear(x, p))
        y.sum().backward()
        torch.testing.assert_close(x.grad, p.detach().sum(0).expand(3, -1))
        p.grad = None
    with torch.no_grad():
        assert torch.equal(model(ids).logits, before)
    held.remove()                                                       # twice is once


def test_generation_within_quantized_weights_leaves_them_in_use():
    model = _model()
    ids = torch.randint(0, 256, (1, 5))
    with quantize_weights(model):
        p = model.layers[0].attn.wqkv
        rows = p.q4
        generate_tokens(model, ids, max_new_tokens=2, weight_bits=4)
        assert p.q4 is rows
    assert not hasattr(p, "q4")


def test_a_model_that_is_split_is_refused_and_gradients_too():
    model = _model()
    whole, model.ex = model.ex, SimpleNamespace(tp_size=2)
    with pytest.raises(ContractError, match="split over tensor-parallel"):
        quantize_weights(model)
    model.ex = whole
    cache = init_kv_cache(model, 1, 8, page_size=4, cache_bits=4)
    ids, at = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(KernelError, match="has no gradient"):
        model.run_with_cache(ids, at, cache)
    with pytest.raises(ContractError, match="cache_bits must be 4 or 16"):
        init_kv_cache(model, 1, 8, cache_bits=3)


def test_sample_command_takes_both(tmp_path, capsys, monkeypatch):
    from research_b200.cli import main

    monkeypatch.chdir(tmp_path)
    raw = tiny_raw_config(tiny_dataset(tmp_path), steps=2, run_id="q4", output_dir=str(tmp_path / "runs"))
    assert main(["run", "train", str(write_toml(raw, tmp_path / "c.toml"))]) == 0
    capsys.readouterr()
    args = ["sample", "checkpoint", str(tmp_path / "runs" / "q4"), "--checkpoint", "latest", "--prompt-ids", "1,2",
            "--max-new-tokens", "3", "--top-k", "1", "--json"]
    assert main(args) == 0
    row = json.loads(capsys.readouterr().out)
    assert "cache_bits" not in row["sampling"]
    assert main([*args, "--cache-bits", "4", "--weight-bits", "4"]) == 0
    row = json.loads(capsys.readouterr().out)
    assert row["sampling"]["cache_bits"] == 4 and row["sampling"]["weight_bits"] == 4 and len(row["generated_ids"]) == 3
    with pytest.raises(SystemExit):
        main([*args, "--cache-bits", "8"])
