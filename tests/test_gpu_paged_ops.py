"""The paged cache operators' kernels against plain 64-bit forms, at the sizes and masks where they can go wrong."""
import pytest
import torch

from lbi_b200 import ops
from paged_oracle import Batch, attention_oracle, check_append, check_attention, check_gather, check_logits
from test_paged_ops import SEQS, refusals

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def clean_status():
    ops.ext().kernel_status(torch.empty(0, device=DEV))
    yield
    assert ops.ext().kernel_status(torch.empty(0, device=DEV)) == 0


# (heads, kv heads, head_dim, page)
SHAPES = [(4, 4, 64, 16), (8, 2, 128, 32), (3, 1, 32, 8), (16, 1, 64, 64), (5, 5, 80, 128), (2, 1, 256, 16)]
STEPS = [(1, 1), (1, 2), (1, 16), (1, 17), (1, 127), (1, 128), (1, 129), (1, 700), (0, 9), (1, 0), (0, 0)]


def test_refusals():
    for i, call in enumerate(refusals(DEV)):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (F16, "same"), (F32, "same"), (BF16, "e4m3"), (F16, "e4m3"), (F32, "e4m3")])
def test_append_and_gather(heads, kv_heads, dim, page, dtype, cache):
    check_append(SEQS, heads, kv_heads, dim, page, dtype, cache, DEV, tail=3, extra_columns=1)
    check_append([(2, 30), (2, 2)], heads, kv_heads, dim, page, dtype, cache, DEV, rope="interleaved", use_cu=False, stride_pad=16)
    check_append([(3, 70)], heads, kv_heads, dim, page, dtype, cache, DEV, rope=None, stride_pad=3)
    batch = Batch(SEQS, heads, kv_heads, dim, page, dtype, cache, DEV, extra_columns=1)
    for max_len in (0, 1, 40, 203):
        check_gather(batch, max_len, dtype)


@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (F32, "e4m3")])
def test_append_of_many_tokens(heads, kv_heads, dim, page, dtype, cache):
    check_append([(333, 401), (0, 5), (312, 312)], heads, kv_heads, dim, page, dtype, cache, DEV, tail=3)


@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (F16, "same"), (F32, "same"), (BF16, "e4m3"), (F16, "e4m3"), (F32, "e4m3")])
def test_single_tokens(heads, kv_heads, dim, page, dtype, cache):
    check_attention(Batch(STEPS, heads, kv_heads, dim, page, dtype, cache, DEV, extra_columns=1), tail=2)


@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (F16, "same"), (F32, "same"), (BF16, "e4m3"), (F16, "e4m3"), (F32, "e4m3")])
def test_a_few_new_tokens(heads, kv_heads, dim, page, dtype, cache):
    check_attention(Batch(SEQS + [(7, 300)], heads, kv_heads, dim, page, dtype, cache, DEV), tail=1)
    check_attention(Batch([(3, 40), (3, 3), (3, 131)], heads, kv_heads, dim, page, dtype, cache, DEV), use_cu=False)


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(2, 2, 64, 16), (4, 1, 64, 32), (3, 1, 128, 8), (2, 1, 128, 128), (2, 1, 80, 64), (2, 1, 64, 128),
                                                       (1, 1, 64, 8)])
@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (F16, "same"), (F32, "same"), (BF16, "e4m3"), (F16, "e4m3")])
def test_chunks_of_new_tokens(heads, kv_heads, dim, page, dtype, cache):
    check_attention(Batch([(130, 130), (1, 50), (129, 400), (0, 3), (64, 64), (200, 100)], heads, kv_heads, dim, page, dtype, cache, DEV), tail=5)


def test_large_scores_and_uneven_values():
    for cache in ("same", "e4m3"):
        check_attention(Batch([(1, 300), (40, 300)], 4, 2, 64, 16, BF16, cache, DEV, spread=8.0), spread=8.0)
        check_attention(Batch([(1, 300)] * 3, 4, 2, 128, 16, F16, cache, DEV, spread=4.0), spread=4.0, scale=1.0)


@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (BF16, "e4m3"), (F32, "same")])
def test_a_long_context(dtype, cache):
    check_attention(Batch([(1, 9000), (1, 37)], 2, 1, 64, 64, dtype, cache, DEV))
    check_attention(Batch([(2, 5000)], 2, 2, 128, 16, dtype, cache, DEV), max_context=100)   # a hint that is too short


@pytest.mark.parametrize("dtype,cache", [(BF16, "same"), (BF16, "e4m3"), (F32, "same")])
def test_many_sequences(dtype, cache):
    """More sequences than a warp looks at in one step, empty ones among them; all heads of a token in several tiles."""
    seqs = [(i % 3, 5 + 7 * i % 60) for i in range(41)]
    check_attention(Batch(seqs, 4, 2, 64, 16, dtype, cache, DEV), tail=1)
    check_append(seqs, 4, 2, 64, 16, dtype, cache, DEV, tail=1)
    check_attention(Batch([(1, 40)] * 35, 2, 1, 64, 16, dtype, cache, DEV), use_cu=False)
    check_attention(Batch([(2, 50), (1, 9)], 40, 1, 64, 16, dtype, cache, DEV))
    check_attention(Batch([(1, 33), (3, 3)], 300, 1, 64, 16, dtype, cache, DEV))


def test_batches_beyond_the_grid_limits_of_one_dimension():
    pages = ops.kv_pages(2, 8, 8, 16, F32, DEV)
    pages.k.normal_()
    table = torch.arange(9000, device=DEV, dtype=torch.int32).remainder(2).view(9000, 1)
    ctx = torch.arange(9000, device=DEV, dtype=torch.int32).remainder(9)
    k, _ = ops.kv_gather(pages, table, ctx, 8)
    want = pages.k[table[:, 0].long()] * (torch.arange(8, device=DEV) < ctx[:, None])[:, None, :, None]
    assert torch.equal(k, want)
    x = torch.randn(70000, 40, device=DEV)
    tokens = torch.arange(70000, device=DEV).remainder(40).view(-1, 1)
    got = ops.adjust_logits(x, tokens, presence=1.0)
    assert torch.equal(got, x.scatter_add(1, tokens, torch.full((70000, 1), -1.0, device=DEV)))


def test_nothing_in_the_table():
    batch = Batch([(1, 0), (2, 1), (0, 0)], 2, 2, 64, 16, BF16, "same", DEV)   # contexts shorter than their new tokens
    check_attention(batch)
    empty = torch.zeros(3, 0, dtype=torch.int32, device=DEV)
    q = batch.queries()
    assert not bool(ops.paged_attention(q, batch.pages, empty, torch.zeros_like(batch.context), 0.1, cu_seqlens=batch.cu).any())
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert not bool(ops.paged_attention(q, batch.pages, empty[:0], none, 0.1, cu_seqlens=zero).any())
    assert ops.paged_attention(q[:0], batch.pages, empty[:0], none, 0.1).shape == (0, 2, 64)


def test_given_outputs_keep_the_rows_behind_the_last_sequence():
    batch = Batch([(2, 20), (1, 5)], 4, 2, 64, 16, BF16, "same", DEV)
    q = batch.queries(tail=2)
    out = torch.full_like(q, 7.0)
    got = ops.paged_attention(q, batch.pages, batch.table, batch.context, 0.125, cu_seqlens=batch.cu, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[3:] == 7.0).all())
    assert torch.equal(out[:3], ops.paged_attention(q, batch.pages, batch.table, batch.context, 0.125, cu_seqlens=batch.cu)[:3])
    qkv = torch.randn(5, 8 * 64, device=DEV).bfloat16()
    out = torch.full_like(q, 7.0)
    ops.kv_append(qkv, batch.pages, batch.table, batch.context, 4, cu_seqlens=batch.cu, out=out)
    assert bool((out[3:] == 7.0).all()) and torch.equal(out[:3], qkv[:3, : 4 * 64].view(3, 4, 64))


def test_strided_and_unaligned_queries():
    batch = Batch([(1, 30), (4, 90)], 4, 2, 64, 16, BF16, "same", DEV)
    q = batch.queries()
    want = ops.paged_attention(q, batch.pages, batch.table, batch.context, 0.125, cu_seqlens=batch.cu)
    wide = torch.zeros(5, 8 * 64 + 8, dtype=BF16, device=DEV)
    for start in (0, 8, 3):
        view = wide[:, start : start + 256].unflatten(1, (4, 64)).copy_(q)
        assert torch.equal(want, ops.paged_attention(view, batch.pages, batch.table, batch.context, 0.125, cu_seqlens=batch.cu))
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(want, ops.paged_attention(turned, batch.pages, batch.table, batch.context, 0.125, cu_seqlens=batch.cu))


def test_results_repeat_bitwise():
    for seqs in ([(1, 3000)] * 3, [(150, 900), (20, 1500)]):
        for cache in ("same", "e4m3"):
            batch = Batch(seqs, 8, 2, 64, 16, BF16, cache, DEV)
            q = batch.queries()
            a, b = (ops.paged_attention(q, batch.pages, batch.table, batch.context, 0.125, cu_seqlens=batch.cu) for _ in range(2))
            assert torch.equal(a, b)


def test_missing_pages_are_skipped_and_recorded():
    like = torch.empty(0, device=DEV)
    for dtype in (BF16, F32):
        pages = ops.kv_pages(2, 8, 1, 64, dtype, DEV)
        table = torch.tensor([[0, 7]], dtype=torch.int32, device=DEV)
        ctx = torch.tensor([10], dtype=torch.int32, device=DEV)
        qkv = torch.randn(10, 3 * 64, device=DEV).to(dtype)
        q = ops.kv_append(qkv, pages, table, ctx, 1)
        assert ops.ext().kernel_status(like) == 84
        assert torch.equal(pages.k[0, 0], qkv[:8, 64:128]) and not bool(pages.k[1].any())
        for rows in (slice(0, 10), slice(9, 10)):
            o = ops.paged_attention(q[rows], pages, table, ctx, 0.1)
            assert ops.ext().kernel_status(like) == 84
            want = torch.softmax(0.1 * qkv[9, :64].double() @ qkv[:8, 64:128].double().t(), -1) @ qkv[:8, 128:].double()
            assert float((o[-1, 0].double() - want).abs().max()) <= (0.02 if dtype == BF16 else 1e-5)
        k, _ = ops.kv_gather(pages, table, ctx, 10)
        assert ops.ext().kernel_status(like) == 84 and not bool(k[0, 0, 8:].any())
        ops.kv_append(qkv, pages, table, ctx, 1, rope=(torch.zeros(4, 32, device=DEV), torch.zeros(4, 32, device=DEV), False))
        assert ops.ext().kernel_status(like) in (83, 84)


@pytest.mark.parametrize("dim,group,cache", [(64, 1, "same"), (128, 3, "same"), (64, 4, "e4m3"), (128, 1, "e4m3")])
def test_chunks_skip_missing_pages_and_cut_long_contexts(dim, group, cache):
    batch = Batch([(150, 1700)], group, 1, dim, 16, BF16, cache, DEV)     # few rows, many keys: cut into parts
    q = batch.queries()
    whole = ops.paged_attention(q, batch.pages, batch.table, batch.context, 0.1)
    batch.table[0, 5] = 10 ** 6
    got = ops.paged_attention(q, batch.pages, batch.table, batch.context, 0.1)
    assert ops.ext().kernel_status(q) == 84
    kept = torch.cat([torch.arange(80), torch.arange(96, 1700)])
    shorter = Batch([(150, 1684)], group, 1, dim, 16, BF16, cache, DEV)
    shorter.k, shorter.v = [batch.k[0][:, kept]], [batch.v[0][:, kept]]
    want, tol = attention_oracle(shorter, q, 0.1)
    assert bool(((got.double().cpu() - want).abs() <= tol).all()) and not torch.equal(got, whole)


@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_any_scale(scale):
    check_attention(Batch([(1, 90), (70, 200)], 2, 2, 64, 16, BF16, "same", DEV), scale=scale)
    check_attention(Batch([(70, 200)], 2, 2, 64, 16, BF16, "e4m3", DEV), scale=scale)


def test_non_finite_rows_of_an_8_bit_cache():
    pages = ops.kv_pages(1, 8, 1, 64, torch.float8_e4m3fn, DEV)
    qkv = torch.randn(3, 3 * 64, device=DEV).bfloat16()
    qkv[0, 64:128], qkv[1, 70] = 0.0, float("nan")
    one = torch.tensor([[0]], dtype=torch.int32, device=DEV)
    ops.kv_append(qkv, pages, one, torch.tensor([3], dtype=torch.int32, device=DEV), 1)
    k, v = ops.kv_gather(pages, one, torch.tensor([3], dtype=torch.int32, device=DEV), 3)
    assert not bool(k[0, 0, 0].any()) and bool(k[0, 0, 1].isnan().all()) and bool(k[0, 0, 2].isfinite().all()) and bool(v.isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("batch,vocab,history", [(1, 1, 1), (2, 31, 7), (3, 4097, 300), (2, 32768, 0), (2, 70001, 999), (5, 8192, 2000)])
def test_logit_rules(dtype, batch, vocab, history):
    check_logits(batch, vocab, history, dtype, DEV)
    check_logits(batch, vocab, history, dtype, DEV, per_row=False, bias="batch", mask="row", stride_pad=5)
    check_logits(batch, vocab, history, dtype, DEV, bias=None, mask=None, prompt=False, lengths=False)


def test_logit_rules_count_a_long_history_and_work_in_place():
    tokens = torch.zeros(1, 70000, dtype=torch.int64, device=DEV)
    tokens[0, ::2] = 3
    x = torch.ones(1, 50, device=DEV)
    out = ops.adjust_logits(x, tokens, presence=1.0, frequency=0.5, out=x)
    assert out.data_ptr() == x.data_ptr()
    want = torch.ones(1, 50, device=DEV)
    want[0, 0] = want[0, 3] = -0.5 * 35000
    assert torch.equal(x, want)


def test_streams_graphs_and_two_calls_at_once():
    """The whole step captured once and replayed with other lengths, next to an eager run on another stream."""
    heads, kv_heads, dim = 8, 2, 64
    pages = [ops.kv_pages(64, 16, kv_heads, dim, torch.float8_e4m3fn, DEV) for _ in range(2)]
    table = torch.arange(64, dtype=torch.int32, device=DEV).view(4, 16)
    ctx = torch.tensor([200, 3, 77, 130], dtype=torch.int32, device=DEV)
    qkv = torch.randn(4, 12 * dim, device=DEV).bfloat16()
    cos, sin = torch.rand(256, 32, device=DEV), torch.rand(256, 32, device=DEV)

    def step(p):
        q = ops.kv_append(qkv, p, table, ctx, heads, rope=(cos, sin, False))
        return ops.paged_attention(q, p, table, ctx, 0.125)

    for p in pages:
        full = torch.randn(200 * 4, 12 * dim, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).bfloat16()
        ops.kv_append(full, p, table, torch.full((4,), 200, dtype=torch.int32, device=DEV), heads)
        step(p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pages[0])
    side = torch.cuda.Stream()
    for lens in ([200, 3, 77, 130], [1, 2, 60, 199]):
        ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        qkv.copy_(torch.randn_like(qkv))
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            eager = step(pages[1])
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("kv_cache", ["paged", "e4m3"])
def test_models_decode_over_pages(kv_cache):
    """A bf16 model's decoder against the forward of the same weights in 64 bits: about ten bf16 roundings per layer and head, half a
    step each, in the relative norm; e4m3 adds half a step of its own to the keys and the values."""
    from lbi_b200.backbones import BackboneSpec
    from lbi_b200.inference import IncrementalDenseDecoder, LogitRules, generate
    from lbi_b200.models import DenseLanguageModel

    torch.manual_seed(0)
    spec = BackboneSpec(name="transformer", dim=256, layers=2, n_heads=4, n_kv_heads=2, d_conv=0)
    model = DenseLanguageModel(vocab_size=500, backbone_spec=spec, tie_embeddings=True).eval().bfloat16()
    ids = torch.randint(0, 500, (2, 230))
    with torch.no_grad():
        want = DenseLanguageModel(vocab_size=500, backbone_spec=spec, tie_embeddings=True).eval().double()
        want.load_state_dict(model.state_dict())
        want = want(ids)
    model = model.to(DEV)
    decoder = IncrementalDenseDecoder(model, 230, kv_cache=kv_cache)
    ids = ids.to(DEV)
    got = torch.cat([decoder.append(ids[:, :200]), decoder.append(ids[:, 200:201]), decoder.append(ids[:, 201:])], dim=1).double().cpu()
    steps = 22 * 2.0 ** -8 + (2 * 2 * 2.0 ** -4 if kv_cache == "e4m3" else 0.0)
    assert float((got - want).norm() / want.norm()) <= steps
    out = generate(model, ids[:, :150], 8, kv_cache=kv_cache, rules=LogitRules(presence_penalty=1e6, allowed_tokens=list(range(100, 400))))
    new = out[:, 150:]
    assert bool(((new >= 100) & (new < 400)).all()) and all(len(set(r)) == 8 for r in new.tolist())
