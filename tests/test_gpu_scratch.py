"""What a call leaves in memory for a later one: the status word of an attention call outlives the scratch of other operators."""
import pytest

pytestmark = pytest.mark.gpu


def attend(bad):
    """A pool that has just attended; with a block id outside the pool in one row where `bad` is set."""
    import torch
    from fused_turboquant_b200 import PagedKVPool
    pool = PagedKVPool(8, 2, 128, 4, 4)
    kv = torch.randn(2, 128, 2, 128, device="cuda").bfloat16()
    pool.store(kv[0], kv[1], torch.arange(128, device="cuda"), layer=0)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1, 2], [0, 1, 99 if bad else 3]], **i32)
    out = pool.shared_attention(torch.randn(2, 8, 128, device="cuda").bfloat16(), table, torch.tensor([40, 41], **i32), 48, torch.tensor([32], **i32))
    assert bool(out.isnan().any()) == bad
    return pool


def use_scratch(name):
    """Calls whose scratch memory reaches far beyond what an attention call of two rows needs."""
    import torch
    from fused_turboquant_b200 import PageTable, beam, logits
    if name == "select":
        assert beam.workspace_bytes(torch.float32, 256, 64, 100, 20) > 2 << 20
        beam.select(torch.randn(256, 64, 100, device="cuda"), torch.zeros(256, 64, device="cuda"), 20)
    elif name == "logits":
        logits.process(torch.randn(60000, 4, 9, device="cuda"))
    else:
        rows, width = 512, 1024
        table = PageTable(rows * width, rows, width, sharing=True)
        table.block_table.copy_(torch.arange(rows * width, dtype=torch.int32, device="cuda").view(rows, width))
        table.seq_lens.fill_(16 * width)
        table.n_free.zero_()
        assert table.fork_workspace_bytes() > 2 << 20
        if name == "fork":
            assert int(table.fork(torch.arange(rows, device="cuda")).done) == 1
        else:
            table.compact()


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("name", ["select", "fork", "compact", "logits"])
def test_the_status_of_attention_outlives_other_operators(name, bad):
    pool = attend(bad)
    use_scratch(name)
    assert pool.decode_status() == int(bad)

