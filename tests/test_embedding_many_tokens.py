"""The embedding's gradient by sorted tokens where the sort takes other forms than for a batch or two: more blocks than each block adds up
by itself, more than one turn of the scan over them, longer chunks, three digits, both together, and a table whose zero rows take longer
pieces.  Against the definition in 64 bits."""

import pytest
import torch

from kareus_amd.backend import get_backend

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]


@pytest.fixture(autouse=True)
def give_memory_back():
    """(Nothing that outlives a test is put into the large pieces that these leave in the allocator.)"""
    yield
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


def ids_of(kind, b, s, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "text":
        ids = (torch.rand(b, s, generator=g) ** 3 * rows).long().clamp_(max=rows - 1)
    elif kind == "one":
        ids = torch.full((b, s), rows - 1)
    elif kind == "padded":
        ids = torch.randint(0, rows, (b, s), generator=g)
        ids[torch.rand(b, s, generator=g) < 0.7] = rows // 2
    else:                                     # "shards": two of three ids belong to others
        ids = torch.randint(-rows, 2 * rows, (b, s), generator=g)
    return ids.cuda()


def check(kind, b, s, h, rows, scale=0.75):
    """Whole in bf16, then added to an fp32 gradient: fp32 sums of n terms, the factor and the sum with what is there, half a step each of
    all the magnitudes, and the store's."""
    be = get_backend("hip")
    ids = ids_of(kind, b, s, rows)
    dout = torch.randn(s, b, h, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    rel = ids.t().reshape(-1)
    keep = (rel >= 0) & (rel < rows)
    flat = dout.view(-1, h).double()[keep]
    # (on the host: half a million additions to one row are atomic ones on the device)
    add = lambda v: torch.zeros(rows, h, dtype=torch.float64).index_add_(0, rel[keep].cpu(), v.cpu()).cuda() * scale  # noqa: E731
    want, mags = add(flat), add(flat.abs())
    count = torch.bincount(rel[keep], minlength=rows)
    got = be.embedding_bwd_sorted(ids, dout, rows, scale=scale)
    roundings = (count + 2)[:, None] * 2.0 ** -24
    assert ((got.double() - want).abs() <= mags * roundings + want.abs() * 2.0 ** -8).all()
    assert not got[count == 0].any() and torch.equal(got, be.embedding_bwd_sorted(ids, dout, rows, scale=scale))
    kept = torch.randn(rows, h, device="cuda")
    before = kept.clone()
    be.embedding_bwd_sorted(ids, dout, rows, scale=scale, out=kept, accumulate=True)
    assert torch.equal(kept[count == 0], before[count == 0])
    assert ((kept.double() - want - before.double()).abs() <= (mags + before.abs()) * roundings).all()


@pytest.mark.parametrize("kind", ["text", "one", "padded", "shards"])
@pytest.mark.parametrize("b,s,h,rows", [(1, 131073, 16, 1000),      # 65 blocks, one token in the last
                                        (3, 60000, 72, 511),        # one digit, 88 blocks
                                        (8, 65600, 8, 32064),       # 257 blocks: two turns of the scan; chunks of 128 tokens
                                        (2, 10007, 40, 300000),     # three digits, few blocks
                                        (5, 30001, 24, 600000)])    # three digits, many blocks
def test_gradient_of_many_tokens(kind, b, s, h, rows):
    check(kind, b, s, h, rows)


def test_gradient_of_more_rows_than_a_launch_has_workgroups():
    """4194304 rows of 8 KB: two rows of zeros to a workgroup."""
    rows, h = 1 << 22, 4096
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB")
    ids = torch.tensor([[0, rows - 1, 7, rows - 1, rows // 2, 3 * rows]], device="cuda")
    dout = torch.randn(6, 1, h, device="cuda").bfloat16()
    got = torch.full((rows, h), 3.0, dtype=torch.bfloat16, device="cuda")
    get_backend("hip").embedding_bwd_sorted(ids, dout, rows, out=got)
    touched = {0: [0], 7: [2], rows // 2: [4], rows - 1: [1, 3]}
    for r, tokens in touched.items():
        assert torch.equal(got[r], sum(dout[t, 0].float() for t in tokens).bfloat16())
        got[r] = 0
    assert all(not part.any() for part in got.view(torch.int16).split(1 << 18))
