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


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 1, 64, 8), (4, 1, 128, 8), (2, 1, 64, 32), (2, 1, 128, 128)])
def test_chunks_whose_last_tile_ends_in_any_word_of_its_mask(heads, kv_heads, dim, page):
    """The slots behind a context hold NaN: a key too many in any of a tile's four words of 32 keys shows in the result."""
    seqs = [(70, 128 + n) for n in (1, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128)]
    check_attention(Batch(seqs, heads, kv_heads, dim, page, BF16, "same", DEV))
