"""The paged cache operators' kernels at the edges of what their documentation allows, against plain 64-bit forms."""
import pytest
import torch

from lbi_b200 import ops
from paged_oracle import Batch, check_attention

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
