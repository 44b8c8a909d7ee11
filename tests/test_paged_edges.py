"""Calls at the edges of what the serving paths document (CPU): what they answer and what they refuse."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from lbi_b200 import ops
from lbi_b200.backbones import BackboneSpec
from lbi_b200.inference import LogitRules, generate
from lbi_b200.models import DenseLanguageModel
from lbi_b200.serve import GenerationService

VOCAB = 50


def dense():
    torch.manual_seed(0)
    spec = BackboneSpec(name="transformer", dim=32, layers=2, n_heads=4, n_kv_heads=2, d_conv=0)
    return DenseLanguageModel(vocab_size=VOCAB, backbone_spec=spec, tie_embeddings=True).eval()


def service():
    return GenerationService(dense(), SimpleNamespace(backbone="transformer", seq_len=32, vocab_size=VOCAB, data_mode="synthetic"))


ASK = {"prompt_ids": [1, 2, 3], "max_new_tokens": 4, "temperature": 0.5}


@pytest.mark.parametrize("bad", [{"presence_penalty": -1e39}, {"presence_penalty": 1e300}, {"frequency_penalty": 1e38},
                                 {"repetition_penalty": 1e-38}, {"repetition_penalty": 1e-320}, {"repetition_penalty": 1e38},
                                 {"logit_bias": {"3": 1e39}}, {"logit_bias": {"3": 1e300}}, {"logit_bias": {"3": float("nan")}}])
def test_rules_that_leave_fp32_are_refused(bad):
    """They would make the softmax of the sampler NaN, which on a GPU ends in a failed assert of the draw."""
    with pytest.raises(ValueError):
        service().handle({**ASK, **bad})


def test_a_bias_tensor_outside_fp32_is_refused():
    with pytest.raises(ValueError):
        generate(dense(), torch.tensor([[1, 2]]), 2, rules=LogitRules(logit_bias=torch.full((VOCAB,), 1e300, dtype=torch.float64)))


@pytest.mark.parametrize("temperature", [0.0, 1e-3, 0.5, 1.0, 1e3])
def test_the_largest_rules_are_sampled_from(temperature):
    top = torch.finfo(torch.float32).max
    s = service()
    ask = {**ASK, "temperature": temperature}
    assert s.handle({**ask, "logit_bias": {"3": 3e38, "4": 2e38}})["new_ids"] == [3] * 4
    assert s.handle({**ask, "logit_bias": {str(i): -top for i in range(VOCAB) if i != 7}})["new_ids"] == [7] * 4
    allowed = [5, 9, 11, 12, 30]
    for extra in ({"logit_bias": {"3": 3e38}}, {"presence_penalty": 1e20}, {"frequency_penalty": -1e20}, {"repetition_penalty": 1e-20},
                  {"repetition_penalty": 1e20, "frequency_penalty": 1e20, "logit_bias": {str(i): -top for i in range(VOCAB)}}):
        assert set(s.handle({**ask, **extra, "allowed_ids": allowed})["new_ids"]) <= set(allowed)


@pytest.mark.parametrize("bad", [float("nan"), 1e-40, 5e-324])
def test_temperatures_that_make_no_distribution_are_refused(bad):
    with pytest.raises(ValueError):
        service().handle({**ASK, "temperature": bad})
    with pytest.raises(ValueError):
        generate(dense(), torch.tensor([[1, 2]]), 2, temperature=bad)


@pytest.mark.parametrize("temperature", [2.0 ** -126, 1e-37, 1e-30, 1e30, float("inf")])
def test_extreme_temperatures_are_sampled_from(temperature):
    """The coldest give the arg-max, the hottest any token that is allowed, beside masked ones, too."""
    s = service()
    ask = {**ASK, "temperature": temperature}
    if temperature < 1:
        for extra in ({}, {"logit_bias": {"3": 50.0, "4": 49.0}}):
            assert s.handle({**ask, **extra})["new_ids"] == s.handle({**ASK, **extra, "temperature": 0.0})["new_ids"]
    allowed = [5, 9, 11, 12, 30]
    assert set(s.handle({**ask, "allowed_ids": allowed})["new_ids"]) <= set(allowed)


@pytest.mark.parametrize("dtype", [torch.bool, torch.int32, torch.float16, torch.bfloat16, torch.float64])
def test_a_bias_tensor_of_any_type(dtype):
    bias = torch.zeros(VOCAB, dtype=dtype)
    bias[7] = 1
    prompt, same = torch.tensor([[1, 2]]), LogitRules(logit_bias=bias.float())
    assert torch.equal(generate(dense(), prompt, 4, rules=LogitRules(logit_bias=bias)), generate(dense(), prompt, 4, rules=same))


def test_an_empty_list_of_allowed_ids_is_refused():
    """It allows nothing; only a missing key (or null) allows everything."""
    s = service()
    with pytest.raises(ValueError):
        s.handle({**ASK, "allowed_ids": []})
    ask = {**ASK, "temperature": 0.0}
    assert s.handle({**ask, "allowed_ids": None})["new_ids"] == s.handle(ask)["new_ids"]
    assert s.handle({**ask, "logit_bias": {}})["new_ids"] == s.handle(ask)["new_ids"]


@pytest.mark.parametrize("bad", [{"allowed_ids": [float("inf")]}, {"logit_bias": {"3": 10 ** 400}}, {"presence_penalty": 10 ** 400}])
def test_numbers_that_do_not_convert_are_malformed_rules(bad):
    with pytest.raises(ValueError):
        service().handle({**ASK, **bad})


class PagedBatch(ctypes.Structure):
    """``lbi_paged_batch`` of api_paged.h."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale", "table", "context", "cu")] + [("table_stride", ctypes.c_int64)] + \
        [(n, ctypes.c_int) for n in ("num_pages", "kv_heads", "page_size", "head_dim", "cache_type", "table_width", "batch", "rows")] + \
        [("status", ctypes.c_void_p)]


class Plan(ctypes.Structure):
    """``lbi_attention_plan`` of api_paged.h."""

    _fields_ = [(n, ctypes.c_int) for n in ("kernel", "rows", "splits", "split_keys")]


F32, BF16, E4M3 = 0, 1, 3


# (sequences, rows, heads, kv heads, head_dim, keys, type, type of the pages): chunks in fp32 and at a head size without tiles of its own,
# many single tokens, drafts of many sequences, a few rows over a long context
@pytest.mark.skipif(not ops.native_available(), reason="the extension is not built")
@pytest.mark.parametrize("batch,rows,heads,kv_heads,dim,keys,kind,cache", [
    (8, 32768, 16, 16, 64, 32768, F32, F32), (1, 4096, 32, 32, 256, 131072, BF16, BF16), (1, 4096, 16, 16, 128, 32768, F32, E4M3),
    (512, 512, 32, 8, 128, 131072, BF16, BF16), (32, 992, 32, 32, 128, 131072, BF16, E4M3), (1, 600, 32, 8, 80, 200000, BF16, BF16),
    (64, 64, 32, 8, 128, 8192, BF16, BF16), (2, 2, 32, 8, 128, 131072, BF16, E4M3), (1, 1, 1, 1, 16, 1 << 30, F32, F32),
    (4, 8192, 16, 16, 64, 10240, BF16, BF16), (1, 256, 2, 2, 64, 65536, BF16, E4M3), (1, 4096, 64, 8, 128, 1 << 20, BF16, BF16)])
def test_the_workspace_of_the_parts_of_a_context_is_bounded(batch, rows, heads, kv_heads, dim, keys, kind, cache):
    plan_of = ctypes.CDLL(ops.ext().__file__).lbi_paged_attention_plan
    plan_of.restype = Plan
    p = PagedBatch(cu=1, kv_heads=kv_heads, page_size=16, head_dim=dim, cache_type=cache, table_width=keys // 16, batch=batch, rows=rows)
    plan = plan_of(ctypes.byref(p), kind, heads, ctypes.c_float(0.1), ctypes.c_int64(0), 148)
    assert plan.splits >= 1 and plan.splits * plan.split_keys >= keys
    assert plan.splits == 1 or rows * heads * plan.splits * (dim + 1) * 4 <= 80 * 2 ** 20


def calls_that_ask_for_gradients(device):
    dtype = torch.bfloat16 if torch.device(device).type == "cuda" else torch.float32
    pages = ops.kv_pages(4, 8, 2, 16, torch.float8_e4m3fn, device)
    table, ctx = torch.zeros(2, 2, dtype=torch.int32, device=device), torch.tensor([3, 4], dtype=torch.int32, device=device)
    qkv, q, cos = torch.zeros(2, 128, dtype=dtype, device=device), torch.zeros(2, 4, 16, dtype=dtype, device=device), torch.zeros(8, 8, device=device)
    for learned in (pages._replace(k_scale=pages.k_scale.clone().requires_grad_()), pages._replace(v_scale=pages.v_scale.clone().requires_grad_())):
        yield lambda p=learned: ops.kv_append(qkv, p, table, ctx, 4)
        yield lambda p=learned: ops.kv_gather(p, table, ctx, 4, dtype=dtype)
        yield lambda p=learned: ops.paged_attention(q, p, table, ctx, 1.0)
    yield lambda: ops.kv_append(qkv, pages, table, ctx, 4, rope=(cos.clone().requires_grad_(), cos, False))
    yield lambda: ops.kv_append(qkv, pages, table, ctx, 4, rope=(cos, cos.clone().requires_grad_(), False))
    yield lambda: ops.kv_append(qkv, pages, table, ctx, 4, out=q.clone().requires_grad_())
    yield lambda: ops.paged_attention(q, pages, table, ctx, 1.0, out=q.clone().requires_grad_())
    x, tokens = torch.zeros(2, 40, device=device), torch.zeros(2, 3, dtype=torch.int64, device=device)
    yield lambda: ops.adjust_logits(x, tokens, out=x.clone().requires_grad_())


def test_every_operand_that_asks_for_a_gradient_is_refused():
    for i, call in enumerate(calls_that_ask_for_gradients("cpu")):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
        with torch.no_grad():
            call()
