"""The embedding gradient of more rows than one row of blocks takes, and of more than any launch takes."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def test_more_blocks_than_a_row_of_them_holds(ctx):
    """A million rows that are one row of whole numbers: every sum is its id's count times the row, exact in float."""
    from brosoundml_amd import tokens
    t, cols, vocab = (1 << 20) - 3, 16392, 5
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-1, vocab, (t,), generator=g).int()
    ids[1000:300000] = 3  # a run over many pieces
    row = torch.randint(-8, 9, (1, cols), generator=g).float()
    dtable = tokens.embedding_bwd(ctx, ids.cuda(), row.bfloat16().cuda().expand(t, cols), vocab)
    count = torch.bincount(ids[ids >= 0], minlength=vocab).float()
    assert float(count.max()) * 8 < 2 ** 24
    assert torch.equal(dtable.cpu(), count[:, None] * row)


def test_what_no_launch_takes_is_refused_before_memory_is_asked_for(ctx):
    """2^30 rows of 2^20 columns: their partial sums would be 140 TB. The refusal names the rows, not the memory."""
    from brosoundml_amd import native, tokens
    ids = torch.zeros(1 << 30, dtype=torch.int32, device="cuda")
    dy = torch.zeros(1, 1 << 20, dtype=torch.bfloat16, device="cuda").expand(1 << 30, 1 << 20)
    held = torch.full((1, 1 << 20), 2.0, device="cuda")
    with pytest.raises(native.KdecError, match="too many tokens"):
        tokens.embedding_bwd(ctx, ids, dy, 1, dtable=held)
    assert (held == 2).all()
