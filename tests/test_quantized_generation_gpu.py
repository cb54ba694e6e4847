"""Generation with a 4-bit cache and 4-bit weights on the GPU."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _trainer(kind="decoder", head_dim=64):
    from research_b200.config import run_spec_from_mapping
    from research_b200.runtime.trainer import Trainer

    model = {"name": kind, "variant": "t", "vocab_size": 512, "hidden_size": 4 * head_dim, "intermediate_size": 512,
             "num_layers": 2, "num_heads": 4, "n_kv_heads": 2, "max_seq_len": 1024, "init": "normal_0.02"}
    if kind == "trinity":
        model["trinity"] = {"initial_dense_layers": 2, "local_window": 48, "local_layers_per_global": 1}
    raw = {"run": {"id": "q4"}, "model": model, "optimizer": {"name": "adamw", "schedule": {"peak_lr": 1e-3}},
           "data": {"train_manifest": "unused.json"},
           "training": {"seq_len": 256, "global_batch_size": 2, "target_tokens": 2 * 256 * 4, "precision": "bf16"}}
    return Trainer(run_spec_from_mapping(raw), build_data=False)


def _dense(pool, B, end, D):
    from research_b200.ops import quantized as q4

    pages = q4.Q4Rows(*(t[0].view(B, -1, *t.shape[2:]) for t in pool))
    return q4.dequantize_rows_reference(pages, D, torch.float64).permute(0, 1, 3, 2, 4).flatten(1, 2)[:, :end]


@pytest.mark.parametrize("D,Hq,H,page", [(128, 4, 2, 128), (64, 6, 2, 20)])
@pytest.mark.parametrize("window", [None, 70])
def test_cache_attends_over_what_it_holds(D, Hq, H, page, window):
    """A prompt, a step, a later piece (its own start not a multiple of 128) and sequences at different places."""

    from research_b200.infer import QuantizedKVCache

    torch.manual_seed(D)
    B = 3
    c = QuantizedKVCache(layers=1, batch=B, max_len=600, kv_heads=H, head_dim=D, page_size=page, dtype=torch.bfloat16,
                         device=torch.device("cuda"))
    at = lambda first, T: (torch.arange(T, dtype=torch.int32, device="cuda") + first).expand(B, T).contiguous()  # noqa: E731
    ragged = at(0, 5) + torch.tensor([[310], [200], [400]], dtype=torch.int32, device="cuda")
    for positions in (at(0, 133), at(133, 1), at(134, 90), at(256, 40), ragged):
        T = positions.shape[1]
        packed = torch.randn(B, T, (Hq + 2 * H) * D, device="cuda").bfloat16()
        q, k, v = (packed[..., a * D:b * D].view(B, T, -1, D) for a, b in ((0, Hq), (Hq, Hq + H), (Hq + H, Hq + 2 * H)))
        got = c.update_and_attend(0, q, k, v, positions, window).double().view(B, T, Hq, D)
        end = int(positions.max()) + 1
        own = int(positions[0, 0]) == 0
        kk, vv = (k.double(), v.double()) if own else (_dense(c.k, B, end, D), _dense(c.v, B, end, D))
        if not own:
            kk, vv = kk.bfloat16().double() if T > 1 else kk, vv.bfloat16().double() if T > 1 else vv
        kk, vv = (t.repeat_interleave(Hq // H, 2) for t in (kk, vv))
        s = torch.einsum("bthd,brhd->bhtr", q.double(), kk) * D ** -0.5
        cols = torch.arange(end, device="cuda")
        seen = cols <= positions[:, :, None]
        if window is not None:
            seen = seen & (cols > positions[:, :, None] - window)
        p = torch.softmax(s.masked_fill(~seen[:, None], float("-inf")), -1)
        want = torch.einsum("bhtr,brhd->bthd", p, vv)
        # bf16 result and bf16 weights in the prompt's kernel, 2^-8 each; scores in fp32 from sums of 128 products: 2^-14
        tol = 2.0 ** -8 * want.abs() + 1.1 * 2.0 ** -8 * torch.einsum("bhtr,brhd->bthd", p, vv.abs())
        assert ((got - want).abs() <= tol + 1e-6).all(), ((got - want).abs() - tol).max()


@pytest.mark.parametrize("kind", ["decoder", "trinity"])
def test_generation_is_repeatable_and_the_graph_is_the_step(kind):
    from research_b200.infer import decode_one, generate_tokens, init_kv_cache, prefill, quantize_weights
    from research_b200.infer.generation import GraphedDecodeStep
    from research_b200.ops import native

    model = _trainer(kind).result.model.eval()
    prompts = torch.randint(0, 512, (3, 130), device="cuda")
    outs = [generate_tokens(model, prompts, max_new_tokens=6, top_k=1, cache_bits=4, weight_bits=4).generated_ids
            for _ in range(2)]
    assert outs[0] == outs[1]
    with quantize_weights(model), torch.no_grad():
        caches = [init_kv_cache(model, 3, 160, cache_bits=4) for _ in range(2)]
        first = [prefill(model, prompts, c) for c in caches]
        assert torch.equal(first[0], first[1])
        token = first[0].argmax(-1)
        before = native.LAUNCHES
        eager = decode_one(model, token, 130, caches[0])
        assert native.LAUNCHES - before >= 2 * 9
        step = GraphedDecodeStep(model, caches[1], token, 130)
        assert torch.equal(step(token, 130), eager)
        nxt = eager.argmax(-1)
        assert torch.equal(step(nxt, 131), decode_one(model, nxt, 131, caches[0]))
        for a, b in zip((*caches[0].k, *caches[0].v), (*caches[1].k, *caches[1].v)):
            assert torch.equal(a, b)
    native.check_status()


def test_logits_with_4_bit_weights_are_those_of_the_weights_they_stand_for():
    from research_b200.infer import init_kv_cache, prefill, quantize_weights
    from research_b200.ops import functional as Fn
    from research_b200.ops import quantized as q4

    model = _trainer().result.model.eval()
    prompts = torch.randint(0, 512, (2, 40), device="cuda")
    with quantize_weights(model), torch.no_grad():
        # 80 rows go through the expanded weights: those of a model that holds them in full, bit for bit
        x = torch.randn(80, 256, device="cuda").bfloat16()
        for layer in model.layers:
            for p in (layer.attn.wqkv, layer.attn.wo, layer.mlp.w_gate_up):
                full = q4.dequantize_rows_q4(p.q4, p.shape[1])
                from research_b200.ops import native

                assert torch.equal(Fn.linear(x, p), native.gemm(x, full.contiguous()))
        got = prefill(model, prompts, init_kv_cache(model, 2, 64, cache_bits=4))
    assert torch.isfinite(got.float()).all()
