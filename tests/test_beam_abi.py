"""What the entry points of a beam search refuse, before anything is launched (no GPU)."""
import numpy as np
import pytest

A = 0x10000        # addresses that nothing follows
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -4


@pytest.fixture(scope="module")
def lib():
    from fused_turboquant_b200 import _lib, build
    build.build()
    return _lib.load()


def call(lib, name, good, **change):
    args = [change.get(k, v) for k, v in good.items()]
    assert not set(change) - set(good), "a misspelt argument"
    return getattr(lib, name)(*args), lib.ftq_last_error().decode()


def at(i):
    return A + (i << 16)


FORK = dict(block_table=at(0), seq_lens=at(1), free_blocks=at(2), n_free=at(3), shares=at(4), n_requests=4, max_blocks=4, num_blocks=8, parents=at(5),
            group=2, keep_lens=None, copies=at(6), done=at(7), workspace=at(8), workspace_bytes=1 << 15, stream=None)
COMPACT = dict(block_table=at(0), seq_lens=at(1), free_blocks=at(2), n_free=at(3), shares=None, n_requests=4, max_blocks=4, num_blocks=8, copies=at(6),
               workspace=at(8), workspace_bytes=1 << 15, stream=None)
LENS = dict(block_table=at(0), seq_lens=at(1), n_groups=2, group=2, max_blocks=4, shared_lens=at(2), stream=None)
COPY = dict(pool=at(0), num_blocks=8, layer_stride=1 << 20, n_layers=2, Hkv=2, head_dim=128, bits_k=4, bits_v=4, copies=at(1), n_copies=3, stream=None)
SELECT = dict(logits=at(0), dtype=2, row_stride=100, n_requests=2, beams=3, vocab=100, scores=at(1), end_tokens=at(2), n_ends=2, n_best=3, out_scores=at(3),
              parents=at(4), tokens=at(5), end_scores=at(6), workspace=at(7), workspace_bytes=1 << 15, stream=None)


@pytest.mark.parametrize("name,good,change,rc,text", [
    ("ftq_pages_fork", FORK, dict(n_requests=8193, group=0), UNSUPPORTED, "8192"),
    ("ftq_pages_fork", FORK, dict(n_requests=-1), INVALID, ""),
    ("ftq_pages_fork", FORK, dict(max_blocks=0), INVALID, "shape"),
    ("ftq_pages_fork", FORK, dict(n_requests=8192, group=0, max_blocks=1 << 18), UNSUPPORTED, "too large"),
    ("ftq_pages_fork", FORK, dict(num_blocks=-1), INVALID, "shape"),
    ("ftq_pages_fork", FORK, dict(group=3), INVALID, "groups of 3"),
    ("ftq_pages_fork", FORK, dict(group=-1), INVALID, "groups of -1"),
    ("ftq_pages_fork", FORK, dict(parents=None), INVALID, "NULL"),
    ("ftq_pages_fork", FORK, dict(shares=None), INVALID, "NULL"),
    ("ftq_pages_fork", FORK, dict(copies=None), INVALID, "NULL"),
    ("ftq_pages_fork", FORK, dict(done=None), INVALID, "NULL"),
    ("ftq_pages_fork", FORK, dict(workspace=None), WORKSPACE, "workspace needs"),
    ("ftq_pages_fork", FORK, dict(workspace_bytes=100), WORKSPACE, "workspace needs"),
    ("ftq_pages_fork", FORK, dict(workspace=at(8) + 8), WORKSPACE, "16-byte"),
    ("ftq_pages_fork", FORK, dict(copies=at(5) + 8), INVALID, "memory of its own"),
    ("ftq_pages_fork", FORK, dict(done=at(5) + 12), INVALID, "memory of its own"),
    ("ftq_pages_fork", FORK, dict(keep_lens=at(6) + 28), INVALID, "memory of its own"),
    ("ftq_pages_fork", FORK, dict(done=at(8) + 64), INVALID, "memory of its own"),
    ("ftq_pages_compact", COMPACT, dict(n_requests=8193), UNSUPPORTED, "8192"),
    ("ftq_pages_compact", COMPACT, dict(copies=None), INVALID, "NULL"),
    ("ftq_pages_compact", COMPACT, dict(copies=at(6) + 4), INVALID, "8-byte"),
    ("ftq_pages_compact", COMPACT, dict(copies=at(2) + 16), INVALID, "memory of its own"),
    ("ftq_pages_compact", COMPACT, dict(workspace_bytes=16), WORKSPACE, "workspace needs"),
    ("ftq_pages_shared_lens", LENS, dict(group=0), INVALID, "shape"),
    ("ftq_pages_shared_lens", LENS, dict(n_groups=-1), INVALID, "shape"),
    ("ftq_pages_shared_lens", LENS, dict(n_groups=1 << 20, group=1 << 12), INVALID, "shape"),
    ("ftq_pages_shared_lens", LENS, dict(shared_lens=None), INVALID, "NULL"),
    ("ftq_pages_shared_lens", LENS, dict(shared_lens=at(1) + 12), INVALID, "memory of its own"),
    ("ftq_copy_pages", COPY, dict(head_dim=96), UNSUPPORTED, "head_dim"),
    ("ftq_copy_pages", COPY, dict(bits_v=5), INVALID, "bits"),
    ("ftq_copy_pages", COPY, dict(n_copies=-1), INVALID, "shape"),
    ("ftq_copy_pages", COPY, dict(Hkv=0), INVALID, "shape"),
    ("ftq_copy_pages", COPY, dict(n_layers=65536), UNSUPPORTED, "layers"),
    ("ftq_copy_pages", COPY, dict(copies=None), INVALID, "NULL"),
    ("ftq_copy_pages", COPY, dict(pool=at(0) + 8), INVALID, "aligned"),
    ("ftq_copy_pages", COPY, dict(layer_stride=(1 << 20) + 8), INVALID, "aligned"),
    ("ftq_beam_select", SELECT, dict(dtype=7), INVALID, "dtype"),
    ("ftq_beam_select", SELECT, dict(beams=0), UNSUPPORTED, "64"),
    ("ftq_beam_select", SELECT, dict(beams=65), UNSUPPORTED, "64"),
    ("ftq_beam_select", SELECT, dict(n_best=65), UNSUPPORTED, "64"),
    ("ftq_beam_select", SELECT, dict(n_best=0), UNSUPPORTED, "64"),
    ("ftq_beam_select", SELECT, dict(n_ends=17), UNSUPPORTED, "16"),
    ("ftq_beam_select", SELECT, dict(vocab=0), INVALID, "shape"),
    ("ftq_beam_select", SELECT, dict(row_stride=99), INVALID, "shape"),
    ("ftq_beam_select", SELECT, dict(n_requests=65536), UNSUPPORTED, "65535"),
    ("ftq_beam_select", SELECT, dict(logits=None), INVALID, "NULL"),
    ("ftq_beam_select", SELECT, dict(logits=at(0) + 1), INVALID, "between"),
    ("ftq_beam_select", SELECT, dict(end_scores=None), INVALID, "NULL"),
    ("ftq_beam_select", SELECT, dict(tokens=at(4) + 4), INVALID, "memory of its own"),
    ("ftq_beam_select", SELECT, dict(out_scores=at(1) + 8), INVALID, "memory of its own"),
    ("ftq_beam_select", SELECT, dict(workspace_bytes=8), WORKSPACE, "workspace needs"),
    ("ftq_beam_select", SELECT, dict(workspace=at(7) + 8), WORKSPACE, "16-byte"),
])
def test_refusals(lib, name, good, change, rc, text):
    got, message = call(lib, name, good, **change)
    assert got == rc and text in message, (got, message)


@pytest.mark.parametrize("change,rc,text", [
    (dict(q_dtype=0), UNSUPPORTED, "16-bit"),
    (dict(group=0), UNSUPPORTED, "1024"),
    (dict(group=1025), UNSUPPORTED, "1024"),
    (dict(head_dim=80), UNSUPPORTED, "head_dim"),
    (dict(Hq=7), INVALID, ""),
    (dict(bits_v=1), INVALID, "bits"),
    (dict(shared_lens=None), INVALID, "NULL"),
    (dict(q=A + 2), INVALID, "aligned"),
    (dict(pool=A + 8), INVALID, "aligned"),
    (dict(max_blocks=3), INVALID, "too narrow"),
    (dict(max_seq_len=-1), INVALID, "shape"),
    (dict(n_requests=1 << 30, group=4), INVALID, "shape"),
    (dict(workspace_bytes=256), WORKSPACE, "workspace needs"),
    (dict(workspace=A + 4), WORKSPACE, "16-byte"),
])
def test_shared_attention_refusals(lib, change, rc, text):
    from fused_turboquant_b200 import _lib
    signs, levels = np.ones(128, np.float32), np.linspace(-2, 2, 16).astype(np.float32)
    need = lib.ftq_shared_workspace_bytes(2, 4, 8, 2, 128, 64)
    assert need > 0
    good = dict(q=A, q_dtype=_lib.BF16, out=A, out_dtype=_lib.BF16, pool=A, num_blocks=8, block_table=A, max_blocks=4, seq_lens=A,
                max_seq_len=64, shared_lens=A, n_requests=2, group=4, Hq=8, Hkv=2, head_dim=128, bits_k=4, bits_v=4,
                levels_k=_lib.fptr(levels), levels_v=_lib.fptr(levels), signs=_lib.fptr(signs), scale=0.1, workspace=A,
                workspace_bytes=need, stream=None)
    got, message = call(lib, "ftq_shared_attn", good, **change)
    assert got == rc and text in message, (got, message)


def test_empty_calls_do_nothing(lib):
    assert call(lib, "ftq_pages_fork", FORK, n_requests=0)[0] == 0
    assert call(lib, "ftq_pages_compact", COMPACT, num_blocks=0)[0] == 0
    assert call(lib, "ftq_pages_shared_lens", LENS, n_groups=0)[0] == 0
    for change in (dict(n_copies=0), dict(n_layers=0), dict(num_blocks=0)):
        assert call(lib, "ftq_copy_pages", COPY, **change)[0] == 0
    assert call(lib, "ftq_beam_select", SELECT, n_requests=0)[0] == 0


def test_workspace_sizes(lib):
    from fused_turboquant_b200 import beam
    import torch
    assert lib.ftq_pages_fork_workspace_bytes(0, 4, 8) == 0
    # the new table, a number per row, two per block
    assert lib.ftq_pages_fork_workspace_bytes(100, 50, 1000) >= 4 * (100 * 50 + 100 + 2 * 1000)
    assert lib.ftq_pages_compact_workspace_bytes(1000) >= 4000
    for bad in ((9, 1, 4, 100, 4, 0), (2, 0, 4, 100, 4, 0), (2, 1, 65, 100, 4, 0), (2, 1, 4, 0, 4, 0), (2, 1, 4, 100, 0, 0), (2, 1, 4, 100, 4, 17)):
        assert lib.ftq_beam_workspace_bytes(*bad) == 0
    assert beam.workspace_bytes(torch.bfloat16, 2, 3, 1000, 4, 2) >= 2 * 3 * (8 + 6 * 8)
    assert beam.workspace_bytes(torch.int32, 2, 3, 1000, 4) == 0
    assert lib.ftq_shared_workspace_bytes(2, 0, 8, 2, 128, 64) == 0
    assert lib.ftq_shared_workspace_bytes(2, 1025, 8, 2, 128, 64) == 0
    assert lib.ftq_shared_workspace_bytes(2, 4, 8, 3, 128, 64) == 0
    a, b = (lib.ftq_shared_workspace_bytes(n, 8, 32, 8, 128, 4096) for n in (1, 64))
    assert 0 < a < b


def test_a_page_table_without_a_device():
    from fused_turboquant_b200 import PageTable
    with pytest.raises(RuntimeError, match="CUDA device"):
        PageTable(8, 2, 2, device="cpu", sharing=True)
