"""Decoding over paged key / value caches and the rules on the logits (CPU): the same results as the training forward."""
import pytest
import torch

from lbi_b200.backbones import BackboneSpec, build_backbone_stack
from lbi_b200.inference import IncrementalDenseDecoder, IncrementalLBIDecoder, LogitRules, generate
from lbi_b200.interfaces import VectorMLPInterface
from lbi_b200.models import DenseLanguageModel, LBILanguageModel
from lbi_b200.serve import GenerationService

VOCAB = 50


def dense(seed=0, **extra):
    torch.manual_seed(seed)
    spec = BackboneSpec(name="transformer", dim=32, layers=2, **{"n_heads": 4, "n_kv_heads": 2, "d_conv": 0, **extra})
    return DenseLanguageModel(vocab_size=VOCAB, backbone_spec=spec, tie_embeddings=True).eval()


def regions(name="transformer", layer_types=None, **extra):
    torch.manual_seed(0)
    spec = BackboneSpec(name=name, dim=32, layers=2 if layer_types is None else len(layer_types), **extra,
                        **({} if layer_types is None else {"layer_types": layer_types}))
    iface = VectorMLPInterface(feature_dim=32, num_regions=4, interface_width=8, interface_map_hidden_dim=16)
    return LBILanguageModel(vocab_size=VOCAB, layers_per_region=1, backbone_spec=spec, interface=iface, region_axis="sequence",
                            num_sequence_regions=4, tie_embeddings=True).eval()


@pytest.mark.parametrize("extra", [dict(d_conv=0), dict(d_conv=4), dict(d_conv=1), dict(d_conv=0, rope_interleaved=True, n_kv_heads=4)])
def test_attention_chunks_equal_the_forward(extra):
    torch.manual_seed(0)
    spec = BackboneSpec(name="transformer", dim=32, layers=1, **{"n_heads": 4, "n_kv_heads": 2, **extra})
    attn = build_backbone_stack(spec).eval().blocks[0].attn
    x = torch.randn(2, 37, 32)
    with torch.no_grad():
        want = attn(x)
    state = attn.allocate_decode_state(2, 37, kv_cache="paged")
    got = torch.cat([attn.extend(x[:, :20], state), attn.step(x[:, 20], state).unsqueeze(1), attn.extend(x[:, 21:23], state), attn.extend(x[:, 23:], state)], 1)
    assert torch.allclose(got, want, atol=5e-6, rtol=1e-5)
    with pytest.raises(ValueError):
        attn.extend(x[:, :1], state)
    eight = attn.allocate_decode_state(2, 37, kv_cache="e4m3")
    got = attn.extend(x, eight)
    assert 0 < float((got - want).norm() / want.norm()) < 2.0 ** -4   # keys and values are half a step of e4m3 off at most
    with pytest.raises(ValueError):
        attn.allocate_decode_state(2, 37, kv_cache="int4")
    with pytest.raises(ValueError):
        attn.extend(x, attn.allocate_decode_state(2, 37))


def test_dense_decoder_over_pages():
    model = dense()
    ids = torch.randint(0, VOCAB, (2, 40))
    with torch.no_grad():
        want = model(ids)
    decoder = IncrementalDenseDecoder(model, 40, kv_cache="paged")
    got = torch.cat([decoder.append(ids[:, :33]), decoder.append(ids[:, 33:34]), decoder.append(ids[:, 34:])], dim=1)
    assert decoder.position == 40 and torch.allclose(got, want, atol=5e-6, rtol=1e-5)
    with pytest.raises(ValueError):
        decoder.append(ids[:, :1])


@pytest.mark.parametrize("name,extra", [("transformer", dict(n_heads=4, n_kv_heads=2, d_conv=4)),
                                        ("hybrid", dict(d_state=16, headdim=16, chunk_size=8, d_conv=4, n_heads=4, layer_types=("mamba2", "transformer")))])
def test_region_decoder_over_pages(name, extra):
    model = regions(name, **extra)
    ids = torch.randint(0, VOCAB, (2, 22))
    with torch.no_grad():
        want, _ = model.forward_with_cache(ids)
    decoder = IncrementalLBIDecoder(model, 22, kv_cache="paged")
    got = torch.cat([decoder.append(ids[:, :4]), decoder.append(ids[:, 4:5]), decoder.append(ids[:, 5:])], dim=1)
    assert torch.allclose(got, want, atol=5e-6, rtol=1e-5)


def test_generation_with_pages_and_refusals():
    model, prompt = dense(), torch.randint(0, VOCAB, (2, 7))
    want = generate(model, prompt, 12)
    assert torch.equal(want, generate(model, prompt, 12, kv_cache="paged"))
    assert generate(model, prompt, 12, kv_cache="e4m3").shape == want.shape
    lbi = regions(n_heads=4, d_conv=0)
    assert torch.equal(generate(lbi, prompt, 9), generate(lbi, prompt, 9, kv_cache="paged"))
    for bad in (lambda: generate(model, prompt, 2, kv_cache="int4"), lambda: generate(lbi, prompt, 2, kv_cache="paged", use_cache=False),
                lambda: generate(model, prompt, 2, kv_cache="paged", use_cache=False)):
        with pytest.raises(ValueError):
            bad()


def test_rules_shape_what_is_generated():
    model, prompt = dense(seed=3), torch.randint(0, VOCAB, (2, 5))
    plain = generate(model, prompt, 10)
    assert torch.equal(plain, generate(model, prompt, 10, rules=LogitRules()))
    only = generate(model, prompt, 10, rules=LogitRules(allowed_tokens=[4, 9]))
    assert set(only[:, 5:].flatten().tolist()) <= {4, 9}
    # a grammar: the next token is the last one plus one
    def follow(tokens):
        mask = torch.zeros(2, VOCAB, dtype=torch.bool)
        return mask.scatter_(1, (tokens[:, -1:] + 1) % VOCAB, True)
    steps = generate(model, prompt, 6, rules=LogitRules(allowed_tokens=follow), kv_cache="paged")
    assert torch.equal(steps[:, 5:], (prompt[:, -1:] + torch.arange(1, 7)) % VOCAB)
    forced = generate(model, prompt, 4, rules=LogitRules(logit_bias={7: 1e4}))
    assert bool((forced[:, 5:] == 7).all())
    fresh = generate(model, prompt[:1], 20, rules=LogitRules(presence_penalty=1e6))     # no token twice
    assert len(set(fresh[0, 5:].tolist())) == 20
    spread = generate(model, prompt[:1], 100, rules=LogitRules(frequency_penalty=1e6))  # every token equally often
    assert sorted(spread[0, 5:].tolist()) == sorted(list(range(VOCAB)) * 2)
    for bad in (dict(repetition_penalty=0.0), dict(presence_penalty=float("nan"))):
        with pytest.raises(ValueError):
            LogitRules(**bad)
    for bad in (dict(logit_bias={VOCAB: 1.0}), dict(logit_bias=torch.zeros(3)), dict(logit_bias=torch.full((VOCAB,), float("-inf"))), dict(allowed_tokens=[VOCAB]), dict(allowed_tokens=[]),
                dict(allowed_tokens=torch.zeros(VOCAB, dtype=torch.bool)), dict(allowed_tokens=lambda t: torch.ones(3, dtype=torch.bool))):
        with pytest.raises(ValueError):
            generate(model, prompt, 2, rules=LogitRules(**bad))


def test_service_takes_the_rules_and_the_cache():
    from types import SimpleNamespace

    cfg = SimpleNamespace(backbone="transformer", seq_len=32, vocab_size=VOCAB, data_mode="synthetic")
    service = GenerationService(dense(), cfg, kv_cache="paged")
    ask = {"prompt_ids": [1, 2, 3], "max_new_tokens": 5}
    assert service.handle(ask)["new_ids"] == GenerationService(dense(), cfg).handle(ask)["new_ids"]
    assert service.handle({**ask, "logit_bias": {"7": 1e4}})["new_ids"] == [7] * 5
    assert set(service.handle({**ask, "allowed_ids": [3, 8], "repetition_penalty": 1.2})["new_ids"]) <= {3, 8}
    for bad in ({"repetition_penalty": -1}, {"logit_bias": {"99": 1}}, {"logit_bias": [1]}, {"allowed_ids": [VOCAB]}, {"presence_penalty": "x"}):
        with pytest.raises(ValueError):
            service.handle({**ask, **bad})
