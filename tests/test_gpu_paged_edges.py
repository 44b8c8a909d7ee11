"""The paged cache operators' kernels at the edges of what their documentation allows, against plain 64-bit forms."""
import pytest
import torch

from lbi_b200 import ops
from lbi_b200.backbones import BackboneSpec
from lbi_b200.backbones.transformer.attention import CausalSelfAttention
from lbi_b200.inference import generate
from lbi_b200.interfaces import VectorMLPInterface
from lbi_b200.models import DenseLanguageModel, LBILanguageModel
from lbi_b200.utils.failure import KernelWaitTimeout
from paged_oracle import Batch, attention_oracle, check_attention
from test_paged_edges import calls_that_ask_for_gradients

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def clean_status():
    ops.ext().kernel_status(torch.empty(0, device=DEV))
    yield
    assert ops.ext().kernel_status(torch.empty(0, device=DEV)) == 0


class Shaped(Batch):
    """A batch with given values: ``make(name, length, generator)`` -> queries, keys or values [heads, length, dim] of a sequence."""

    def __init__(self, make, seqs, *args, **kw):
        self.make, self.made = make, 0
        super().__init__(seqs, *args, **kw)

    def _values(self, n, spread):
        self.made += 1   # the keys of all sequences, then the values
        return self.make("k" if self.made <= len(self.seqs) else "v", n, self.gen).to(self.dtype).double()

    def queries(self, tail=0, spread=1.0):
        return torch.cat([self.make("q", new, self.gen).transpose(0, 1) for new, _ in self.seqs]).to(self.dtype).to(self.device)


# (new tokens, heads of one kv head, head_dim): tiles of 8 and of 16 rows, of 256 rows
ROW_FORMS = [(1, 1, 32), (1, 1, 64), (1, 1, 128), (3, 4, 32), (3, 4, 64), (3, 4, 128)]
TILE_FORMS = [(100, 1, 64), (100, 1, 128)]
TYPES = [(BF16, "same"), (F16, "same"), (BF16, "e4m3"), (F16, "e4m3")]


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 1, 64, 8), (4, 1, 128, 8), (2, 1, 64, 32), (2, 1, 128, 128)])
def test_chunks_whose_last_tile_ends_in_any_word_of_its_mask(heads, kv_heads, dim, page):
    """The slots behind a context hold NaN: a key too many in any of a tile's four words of 32 keys shows in the result."""
    seqs = [(70, 128 + n) for n in (1, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128)]
    check_attention(Batch(seqs, heads, kv_heads, dim, page, BF16, "same", DEV))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("new,group,dim,binades,keys,at", [(*f, 24.5, 6000, at) for f in ROW_FORMS + TILE_FORMS for at in (0, 2500)]
                         + [(*f, 28.0, 12000, 0) for f in ROW_FORMS])
def test_one_key_far_above_thousands_of_others(new, group, dim, dtype, cache, binades, keys, at):
    """The heavy key's values are 0 but for one element, so the other elements are the small weights' alone.  Every weight is still a
    normal fp16 number (2^-24.5 or 2^-28, times 2^11 or 2^15): the tolerance's half step per weight holds."""
    def make(name, n, gen):
        x = torch.zeros(group if name == "q" else 1, n, dim)
        if name == "q":
            x[..., 0] = 4.0
        elif name == "k":
            x[:, at : at + 1, 0] = binades * 0.6931471805599453 / 4.0
        else:
            x[:] = 64.0 + 16.0 * torch.rand(1, n, dim, generator=gen)
            x[:, at : at + 1] = 0.0
            x[:, at : at + 1, 1] = 64.0
        return x
    # the short hint keeps the context in one part
    check_attention(Shaped(make, [(new, keys)], group, 1, dim, 64, dtype, cache, DEV), scale=1.0, max_context=64)


# (new tokens, type, head_dim): every kernel, whole and in parts of a long context
KERNELS = [(1, BF16, 64), (6, BF16, 64), (100, BF16, 64), (100, BF16, 128), (3, F32, 64), (2, BF16, 80)]


@pytest.mark.parametrize("new,dtype,dim", KERNELS)
@pytest.mark.parametrize("keys", [200, 3000])
def test_rows_in_front_of_the_first_sequence_belong_to_nobody(new, dtype, dim, keys):
    batch = Batch([(new, keys), (new, new)], 2, 1, dim, 16, dtype, "same", DEV)
    front, behind, n = 5, 2, 2 * new
    q = torch.ones(front + n + behind, 2, dim, device=DEV, dtype=dtype)
    q[front : front + n] = batch.queries()
    call = dict(q=q, pages=batch.pages, page_table=batch.table, context_lens=batch.context, scale=0.125, cu_seqlens=batch.cu + front)
    want = ops.paged_attention(**{**call, "q": q[front : front + n], "cu_seqlens": batch.cu})
    nan = [torch.full((2 ** i,), float("nan"), device=DEV) for i in range(8, 24)]   # what new memory holds
    del nan
    got = ops.paged_attention(**call)
    assert torch.equal(got[front : front + n], want)
    assert bool((got[:front] == 0).all()) and bool((got[front + n :] == 0).all())
    out = torch.full_like(q, 7.0)
    ops.paged_attention(**call, out=out)
    assert torch.equal(out[front : front + n], want)
    assert bool((out[:front] == 7).all()) and bool((out[front + n :] == 7).all())


def test_append_leaves_rows_in_front_of_the_first_sequence_alone():
    batch = Batch([(2, 20), (1, 5)], 4, 2, 64, 16, BF16, "same", DEV)
    qkv = torch.randn(9, 8 * 64, device=DEV).bfloat16()
    got = ops.kv_append(qkv, batch.pages, batch.table, batch.context, 4, cu_seqlens=batch.cu + 3)
    assert torch.equal(got[3:6], qkv[3:6, : 4 * 64].view(3, 4, 64)) and not bool(got[:3].any()) and not bool(got[6:].any())
    out = torch.full_like(got, 7.0)
    ops.kv_append(qkv, batch.pages, batch.table, batch.context, 4, cu_seqlens=batch.cu + 3, out=out)
    assert torch.equal(out[3:6], got[3:6]) and bool((out[:3] == 7).all()) and bool((out[6:] == 7).all())


@pytest.mark.parametrize("new,dtype,dim", KERNELS)
@pytest.mark.parametrize("keys", [200, 3000])
def test_a_context_that_outruns_its_table_is_recorded(new, dtype, dim, keys):
    """Positions behind the table are skipped: the result is that of the keys that have a page."""
    batch = Batch([(new, keys)], 2, 1, dim, 8, dtype, "same", DEV)
    q = batch.queries()
    ops.paged_attention(q, batch.pages, batch.table, batch.context, 0.125)
    assert ops.ext().kernel_status(q) == 0
    columns = (keys - new) // 8 - 2                       # every new token sees all keys that are left
    got = ops.paged_attention(q, batch.pages, batch.table[:, :columns].contiguous(), batch.context, 0.125)
    assert ops.ext().kernel_status(q) == 84
    left = Batch([(1, columns * 8)], 2, 1, dim, 8, dtype, "same", DEV)
    left.k, left.v = ([x[0][:, : columns * 8]] for x in (batch.k, batch.v))
    for i in range(new):
        want, tol = attention_oracle(left, q[i : i + 1], 0.125)
        assert bool(((got[i : i + 1].double().cpu() - want).abs() <= tol).all())


def test_every_operand_that_asks_for_a_gradient_is_refused():
    for i, call in enumerate(calls_that_ask_for_gradients(DEV)):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
        with torch.no_grad():
            call()


def test_a_bias_or_a_mask_without_dimensions_is_refused():
    x, tokens = torch.zeros(2, 40, device=DEV), torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    for bad in (dict(bias=torch.zeros((), device=DEV)), dict(allowed=torch.zeros((), dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            ops.adjust_logits(x, tokens, **bad)


def test_histories_whose_steps_would_leave_32_bits_are_refused():
    with pytest.raises(ValueError):
        ops.adjust_logits(torch.zeros(1, 40, device=DEV), torch.empty(1, 2 ** 31 - 1000, dtype=torch.int64, device=DEV))


def test_tables_whose_positions_would_leave_32_bits_are_refused():
    pages = ops.kv_pages(2, 128, 1, 64, BF16, DEV)
    table = torch.zeros(1, 2 ** 24 - 1, dtype=torch.int32, device=DEV)     # 2^31 - 128 positions
    ctx = torch.ones(1, dtype=torch.int32, device=DEV)
    qkv, q = torch.zeros(1, 3 * 64, device=DEV).bfloat16(), torch.zeros(1, 1, 64, device=DEV).bfloat16()
    for call in (lambda: ops.kv_append(qkv, pages, table, ctx, 1), lambda: ops.kv_gather(pages, table, ctx, 4),
                 lambda: ops.paged_attention(q, pages, table, ctx, 1.0)):
        with pytest.raises(ValueError):
            call()


def dense_model(dtype=BF16):
    torch.manual_seed(0)
    spec = BackboneSpec(name="transformer", dim=128, layers=2, n_heads=4, n_kv_heads=2, d_conv=0)
    return DenseLanguageModel(vocab_size=300, backbone_spec=spec, tie_embeddings=True).eval().to(dtype).to(DEV)


def region_model(dtype=BF16):
    torch.manual_seed(0)
    spec = BackboneSpec(name="transformer", dim=128, layers=2, n_heads=4, n_kv_heads=2, d_conv=0)
    interface = VectorMLPInterface(feature_dim=128, num_regions=2, interface_width=8, interface_map_hidden_dim=16)
    return LBILanguageModel(vocab_size=300, layers_per_region=1, backbone_spec=spec, interface=interface, region_axis="sequence",
                            num_sequence_regions=2, tie_embeddings=True).eval().to(dtype).to(DEV)


@pytest.mark.parametrize("build", [dense_model, region_model])
def test_generation_raises_what_the_kernels_recorded(build, monkeypatch):
    model, prompt = build(), torch.randint(0, 300, (2, 40), device=DEV)
    want = generate(model, prompt, 4, kv_cache="paged")
    allocate = CausalSelfAttention.allocate_decode_state

    def without_a_page(self, *args, **kw):
        state = allocate(self, *args, **kw)
        state["table"][1, 1] = 10 ** 6      # no such page: the operators skip it and record that
        return state

    monkeypatch.setattr(CausalSelfAttention, "allocate_decode_state", without_a_page)
    with pytest.raises(KernelWaitTimeout, match="84"):
        generate(model, prompt, 4, kv_cache="paged")
    monkeypatch.undo()
    assert torch.equal(generate(model, prompt, 4, kv_cache="paged"), want)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("group,dim", [(1, 64), (4, 64), (1, 128), (4, 128)])
def test_scores_that_grow_along_the_context(group, dim, dtype, cache):
    """By 18 binades per 128 keys: the running maximum moves and the output is rescaled in every tile of every kernel."""
    def make(name, n, gen):
        x = 0.25 * torch.randn(group if name == "q" else 1, n, dim, generator=gen)
        if name == "q":
            x[..., 0] = 4.0
        elif name == "k":
            x[..., 0] = torch.arange(n) / 40.0
        return x
    for seqs in ([(130, 700), (100, 900)], [(1, 1500), (1, 300)], [(3, 700)]):
        check_attention(Shaped(make, seqs, group, 1, dim, 16, dtype, cache, DEV), scale=1.0)


@pytest.mark.parametrize("dtype,cache", [*TYPES, (F32, "e4m3")])
@pytest.mark.parametrize("new,group,dim", ROW_FORMS + TILE_FORMS + [(100, 4, 128)])
def test_values_whose_size_differs_from_token_to_token(new, group, dim, dtype, cache):
    """By up to 2^10, and every fifth token's are 0: the weights of an 8-bit cache carry the scales of the values."""
    def make(name, n, gen):
        x = torch.randn(group if name == "q" else 1, n, dim, generator=gen)
        if name == "v":
            x = x * 2.0 ** torch.randint(-8, 3, (1, n, 1), generator=gen)
            x[:, ::5] = 0.0
        return x
    check_attention(Shaped(make, [(new, 700), (new, new), (new, 1200)], group, 1, dim, 16, dtype, cache, DEV))


@pytest.mark.parametrize("build", [dense_model, region_model])
@pytest.mark.parametrize("kv_cache", ["paged", "e4m3"])
def test_models_in_fp32_decode_as_on_the_host(build, kv_cache):
    """The same weights through the kernels and through the statements.  Sums of at most 2700 terms follow one another, half a step of
    fp32 each; in 8 bits a code near the middle of two may round the other way, an eighth of one of 2^17 elements: 64 of those are
    2^-3 sqrt(64 / 2^17) of the norm."""
    from lbi_b200.inference import IncrementalDenseDecoder, IncrementalLBIDecoder

    model = build(F32)
    ids = torch.randint(0, 300, (2, 230), generator=torch.Generator().manual_seed(1))
    decoder = IncrementalDenseDecoder if build is dense_model else IncrementalLBIDecoder
    rows = []
    for device in (DEV, "cpu"):
        d = decoder(model.to(device), 230, kv_cache=kv_cache)
        x = ids.to(device)
        rows.append(torch.cat([d.append(x[:, :200]), d.append(x[:, 200:201]), d.append(x[:, 201:])], dim=1).double().cpu())
    assert float((rows[0] - rows[1]).norm() / rows[1].norm()) <= 2700 * 2.0 ** -24 + (2.0 ** -3 * (64 / 2 ** 17) ** 0.5 if kv_cache == "e4m3" else 0.0)


FIRST_CALL_IN_A_CAPTURE = """
import torch
from lbi_b200 import ops

dev, bf16 = "cuda", torch.bfloat16
pages = ops.KVPages(*(torch.randn(2, 1, 8, 64, device=dev, dtype=bf16) for _ in range(2)))     # not from kv_pages
table = torch.tensor([[0, 1]], dtype=torch.int32, device=dev)
context = torch.tensor([10], dtype=torch.int32, device=dev)
q = torch.randn(1, 1, 64, device=dev, dtype=bf16)
junk = [torch.full((2 ** i,), 7, dtype=torch.int32, device=dev) for i in range(20)]
del junk
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = ops.paged_attention(q, pages, table, context, 0.125)
assert ops.ext().kernel_status(q) == 0, "before the first replay"
graph.replay()
assert ops.ext().kernel_status(q) == 0
want = ops.paged_attention(q, pages, table, context, 0.125)
assert torch.equal(out, want)
table[0, 1] = 9
graph.replay()
table[0, 1] = 1
graph.replay()
assert ops.ext().kernel_status(q) == 84, "a record is kept until it is read"
table[0, 1] = 9
ops.paged_attention(q, pages, table, context, 0.125)
table[0, 1] = 1
graph.replay()
assert ops.ext().kernel_status(q) == 84, "an eager call's, too"
assert ops.ext().kernel_status(q) == 0
"""


def test_records_outlive_replays_when_the_first_call_was_captured():
    import subprocess
    import sys

    done = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
