"""The paged cache operators on CPU tensors (their PyTorch statements) against plain 64-bit forms, and what they refuse."""
import pytest
import torch

from lbi_b200 import ops
from paged_oracle import Batch, check_append, check_attention, check_gather, check_logits

SEQS = [(1, 1), (3, 3), (0, 5), (2, 17), (5, 40), (0, 0), (4, 2)]   # the last: two rows before position 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_statements_match_the_formulas(dtype, cache):
    check_attention(Batch(SEQS, 6, 2, 24, 8, dtype, cache, extra_columns=2), tail=2)
    check_append(SEQS, 3, 1, 24, 8, dtype, cache, "cpu", tail=2, extra_columns=1)
    check_append([(2, 9), (2, 2)], 2, 2, 16, 16, dtype, cache, "cpu", rope="interleaved", use_cu=False)
    check_append([(1, 4)], 2, 2, 16, 16, dtype, cache, "cpu", rope=None)
    check_gather(Batch(SEQS, 6, 2, 24, 8, dtype, cache), 40, dtype)
    check_gather(Batch(SEQS, 6, 2, 24, 8, dtype, cache), 11, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias,mask", [("row", "batch"), ("batch", "row"), (None, None)])
def test_logit_rules_statement(dtype, bias, mask):
    check_logits(3, 101, 40, dtype, "cpu", bias=bias, mask=mask)
    check_logits(2, 33, 5, dtype, "cpu", per_row=False, bias=bias, mask=mask, prompt=False, lengths=False)
    check_logits(1, 64, 0, dtype, "cpu", bias=bias, mask=mask)


def test_token_mask_words():
    mask = torch.zeros(2, 70, dtype=torch.bool)
    mask[0, 0] = mask[0, 31] = mask[1, 32] = mask[1, 69] = True
    words = ops.pack_token_mask(mask)
    assert words.dtype == torch.int32 and words.tolist() == [[1 - 2 ** 31, 0, 0], [0, 1, 32]]
    with pytest.raises(ValueError):
        ops.pack_token_mask(mask.int())


def test_append_then_attend_equals_attention_over_the_whole_sequence():
    torch.manual_seed(0)
    heads, kv_heads, dim, n = 4, 2, 16, 21
    qkv = torch.randn(n, (heads + 2 * kv_heads) * dim)
    pages = ops.kv_pages(4, 8, kv_heads, dim, torch.float32)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    outs, done = [], 0
    for new in (5, 1, 1, 9, 5):
        done += new
        ctx = torch.tensor([done], dtype=torch.int32)
        q = ops.kv_append(qkv[done - new : done], pages, table, ctx, heads)
        outs.append(ops.paged_attention(q, pages, table, ctx, 0.25))
    q, k, v = (t.view(n, -1, dim).transpose(0, 1) for t in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1))
    want = torch.nn.functional.scaled_dot_product_attention(q, k.repeat_interleave(2, 0), v.repeat_interleave(2, 0), is_causal=True, scale=0.25)
    assert torch.allclose(torch.cat(outs), want.transpose(0, 1), atol=1e-5)


def refusals(device):
    """Calls that every device refuses with ValueError (shared with the GPU tests)."""
    dt = torch.bfloat16 if torch.device(device).type == "cuda" else torch.float32
    pages = ops.kv_pages(4, 8, 2, 16, dt, device)
    table = torch.zeros(2, 2, dtype=torch.int32, device=device)
    ctx = torch.tensor([3, 4], dtype=torch.int32, device=device)
    qkv = torch.zeros(2, 8 * 16, dtype=dt, device=device)
    q = torch.zeros(2, 4, 16, dtype=dt, device=device)
    other = torch.float16
    e4m3 = ops.kv_pages(4, 8, 2, 16, torch.float8_e4m3fn, device)
    cos = torch.zeros(8, 8, device=device)
    logits, tokens = torch.zeros(2, 40, dtype=dt, device=device), torch.zeros(2, 3, dtype=torch.int64, device=device)
    yield lambda: ops.kv_pages(4, 12, 2, 16, dt, device)
    yield lambda: ops.kv_pages(4, 8, 2, 16, torch.int8, device)
    yield lambda: ops.kv_pages(0, 8, 2, 16, dt, device)
    yield lambda: ops.kv_append(qkv[:, :-16], pages, table, ctx, 4)                                   # columns
    yield lambda: ops.kv_append(qkv.to(other), pages, table, ctx, 4)                                  # type of the pages
    yield lambda: ops.kv_append(qkv, pages, table.long(), ctx, 4)                                     # int64 table
    yield lambda: ops.kv_append(qkv, pages, table[:1], ctx, 4)                                        # rows of the table
    yield lambda: ops.kv_append(qkv, pages, table, ctx, 4, cu_seqlens=ctx)                            # entries of cu_seqlens
    yield lambda: ops.kv_append(qkv[:1], pages, table, ctx, 4)                                        # uneven rows
    yield lambda: ops.kv_append(qkv, pages, table, ctx, 4, rope=(cos[:, :4], cos[:, :4], False))      # width of the rotary table
    yield lambda: ops.kv_append(qkv, pages, table, ctx, 4, rope=(cos.double(), cos.double(), False))  # type of the rotary table
    yield lambda: ops.kv_append(qkv, e4m3._replace(k_scale=None), table, ctx, 4)                      # 8-bit pages without scales
    yield lambda: ops.kv_append(qkv, pages._replace(v=pages.v[:2]), table, ctx, 4)                    # k and v differ
    yield lambda: ops.kv_append(qkv, pages, table, ctx, 4, out=q[:1])
    yield lambda: ops.kv_append(qkv.clone().requires_grad_(), pages, table, ctx, 4)
    yield lambda: ops.paged_attention(q[:, :3], pages, table, ctx, 1.0)                               # heads
    yield lambda: ops.paged_attention(q[:, :, :8], pages, table, ctx, 1.0)                            # head_dim
    yield lambda: ops.paged_attention(q.to(other), pages, table, ctx, 1.0)
    yield lambda: ops.paged_attention(q, pages, table, ctx.long(), 1.0)
    yield lambda: ops.paged_attention(q, pages, table, ctx, 1.0, out=q.half())
    yield lambda: ops.paged_attention(q.clone().requires_grad_(), pages, table, ctx, 1.0)
    yield lambda: ops.kv_gather(pages, table, ctx, -1)
    yield lambda: ops.kv_gather(pages, table, ctx, 4, dtype=other)
    yield lambda: ops.kv_gather(e4m3, table, ctx, 4, dtype=torch.int8)
    yield lambda: ops.adjust_logits(logits[0], tokens)
    yield lambda: ops.adjust_logits(logits, tokens.int())
    yield lambda: ops.adjust_logits(logits, tokens[:1])
    yield lambda: ops.adjust_logits(logits, tokens, repetition=0.0)
    yield lambda: ops.adjust_logits(logits, tokens, presence=torch.zeros(3, device=device))
    yield lambda: ops.adjust_logits(logits, tokens, lengths=torch.zeros(2, dtype=torch.int64, device=device))
    yield lambda: ops.adjust_logits(logits, tokens, bias=torch.zeros(39, device=device))
    yield lambda: ops.adjust_logits(logits, tokens, allowed=torch.zeros(2, 1, dtype=torch.int32, device=device))
    yield lambda: ops.adjust_logits(logits, tokens, out=torch.zeros(2, 39, device=device))
    # one table of the two, and gradients that an operand other than the rows asks for
    yield lambda: ops.kv_append(qkv, pages, table, ctx, 4, rope=(cos, None, False))
    yield lambda: ops.kv_append(qkv, pages, table, ctx, 4, rope=(None, cos, False))
    learned = pages._replace(v=pages.v.clone().requires_grad_())
    yield lambda: ops.kv_append(qkv, learned, table, ctx, 4)
    yield lambda: ops.paged_attention(q, learned, table, ctx, 1.0)
    yield lambda: ops.kv_gather(learned, table, ctx, 4)
    yield lambda: ops.adjust_logits(logits, tokens, frequency=torch.zeros(2, device=device, requires_grad=True))
    yield lambda: ops.adjust_logits(logits, tokens, bias=torch.zeros(40, device=device, requires_grad=True))


def test_refusals():
    for i, call in enumerate(refusals("cpu")):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_missing_pages_are_skipped():
    pages = ops.kv_pages(2, 8, 1, 16, torch.float32)
    table = torch.tensor([[0, 7]], dtype=torch.int32)     # the second page does not exist
    ctx = torch.tensor([10], dtype=torch.int32)
    qkv = torch.randn(10, 3 * 16)
    q = ops.kv_append(qkv, pages, table, ctx, 1)
    assert torch.equal(pages.k[0, 0], qkv[:8, 16:32]) and not bool(pages.k[1].any())
    o = ops.paged_attention(q, pages, table, ctx, 1.0)
    want = torch.softmax(qkv[9, :16] @ qkv[:8, 16:32].t(), -1) @ qkv[:8, 32:]
    assert torch.allclose(o[9, 0], want, atol=1e-5)
    k, _ = ops.kv_gather(pages, table, ctx, 10)
    assert not bool(k[0, 0, 8:].any())
