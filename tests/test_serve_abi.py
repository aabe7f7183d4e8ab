"""What the entry points of a step with drafted trees refuse, before anything is launched (no GPU)."""
import ctypes

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


EXTEND = dict(block_table=A, seq_lens=A, free_blocks=A, n_free=A, n_requests=2, max_blocks=4, num_blocks=8, new_lens=A, width=4, packed=0,
              slots=A, granted=A, starts=A, stream=None)
TRIM = dict(block_table=A, seq_lens=A, free_blocks=A, n_free=A, n_requests=2, max_blocks=4, num_blocks=8, keep_lens=A, stream=None)
MASKS = dict(parents=A, tree_lens=None, context_lens=None, B=2, n_nodes=8, masks=A, positions=A, stream=None)
COMMIT = dict(pool=A, num_blocks=8, layer_stride=1 << 20, n_layers=2, block_table=A, max_blocks=4, seq_lens=A, tree_lens=None, tokens=A,
              parents=A, next_tokens=A, B=2, n_nodes=8, Hkv=2, head_dim=128, bits_k=4, bits_v=4, path=A, n_accepted=A, out_tokens=A,
              new_lens=A + 64, stream=None)
LOGITS = dict(logits=A, dtype=2, row_stride=100, n_requests=2, rows=3, vocab=100, history=None, history_stride=0, history_lens=None,
              prompt_lens=None, repetition=None, frequency=None, presence=None, bias_ids=None, bias=None, n_bias=0, allowed=None,
              allowed_stride=0, tree_tokens=None, tree_masks=None, out=A << 8, best=None, workspace=None, workspace_bytes=0, stream=None)


@pytest.mark.parametrize("name,good,change,rc,text", [
    ("ftq_pages_extend", EXTEND, dict(n_requests=8193), UNSUPPORTED, "8192"),
    ("ftq_pages_extend", EXTEND, dict(n_requests=-1), INVALID, ""),
    ("ftq_pages_extend", EXTEND, dict(max_blocks=0), INVALID, ""),
    ("ftq_pages_extend", EXTEND, dict(num_blocks=-1), INVALID, ""),
    ("ftq_pages_extend", EXTEND, dict(width=-1), INVALID, "width"),
    ("ftq_pages_extend", EXTEND, dict(width=1 << 30), INVALID, "width"),
    ("ftq_pages_extend", EXTEND, dict(slots=None), INVALID, "NULL"),
    ("ftq_pages_extend", EXTEND, dict(block_table=None), INVALID, "NULL"),
    ("ftq_pages_trim", TRIM, dict(keep_lens=None), INVALID, "NULL"),
    ("ftq_pages_trim", TRIM, dict(n_requests=8193), UNSUPPORTED, "8192"),
    ("ftq_tree_masks", MASKS, dict(n_nodes=0), UNSUPPORTED, "256"),
    ("ftq_tree_masks", MASKS, dict(n_nodes=257), UNSUPPORTED, "256"),
    ("ftq_tree_masks", MASKS, dict(B=-1), INVALID, "B=-1"),
    ("ftq_tree_masks", MASKS, dict(positions=None), INVALID, "NULL"),
    ("ftq_tree_commit", COMMIT, dict(head_dim=96), UNSUPPORTED, "head_dim"),
    ("ftq_tree_commit", COMMIT, dict(bits_k=5), INVALID, "bits"),
    ("ftq_tree_commit", COMMIT, dict(n_nodes=300), UNSUPPORTED, "256"),
    ("ftq_tree_commit", COMMIT, dict(n_layers=0), INVALID, "layers"),
    ("ftq_tree_commit", COMMIT, dict(path=None), INVALID, "NULL"),
    ("ftq_tree_commit", COMMIT, dict(pool=A + 8), INVALID, "aligned"),
    ("ftq_tree_commit", COMMIT, dict(layer_stride=(1 << 20) + 8), INVALID, "aligned"),
    ("ftq_tree_commit", COMMIT, dict(new_lens=A), INVALID, "memory of their own"),
    ("ftq_logits_process", LOGITS, dict(dtype=7), INVALID, "dtype"),
    ("ftq_logits_process", LOGITS, dict(vocab=0), INVALID, "shape"),
    ("ftq_logits_process", LOGITS, dict(row_stride=99), INVALID, "shape"),
    ("ftq_logits_process", LOGITS, dict(rows=65536), UNSUPPORTED, "65535"),
    ("ftq_logits_process", LOGITS, dict(out=None), INVALID, "nothing to write"),
    ("ftq_logits_process", LOGITS, dict(history=A), INVALID, "history_lens"),
    ("ftq_logits_process", LOGITS, dict(n_bias=2, bias_ids=A), INVALID, "ids and values"),
    ("ftq_logits_process", LOGITS, dict(tree_tokens=A), INVALID, "tokens and masks"),
    ("ftq_logits_process", LOGITS, dict(tree_tokens=A, tree_masks=A, rows=257), UNSUPPORTED, "256"),
    ("ftq_logits_process", LOGITS, dict(allowed=A, allowed_stride=3), INVALID, "words"),
    ("ftq_logits_process", LOGITS, dict(out=A), INVALID, "overlaps"),
    ("ftq_logits_process", LOGITS, dict(best=A), WORKSPACE, "workspace needs"),
])
def test_refusals(lib, name, good, change, rc, text):
    got, message = call(lib, name, good, **change)
    assert got == rc and text in message, (got, message)


@pytest.mark.parametrize("change,rc,text", [
    (dict(q_dtype=0), UNSUPPORTED, "16-bit"),
    (dict(n_nodes=0), UNSUPPORTED, "256"),
    (dict(n_nodes=257), UNSUPPORTED, "256"),
    (dict(head_dim=80), UNSUPPORTED, "head_dim"),
    (dict(Hq=7), INVALID, ""),
    (dict(bits_v=1), INVALID, "bits"),
    (dict(masks=None), INVALID, "NULL"),
    (dict(q=A + 2), INVALID, "aligned"),
    (dict(pool=A + 8), INVALID, "aligned"),
    (dict(max_blocks=3), INVALID, "too narrow"),
    (dict(max_seq_len=-1), INVALID, "shape"),
    (dict(workspace_bytes=256), WORKSPACE, "workspace needs"),
    (dict(workspace=A + 4), WORKSPACE, "16-byte"),
])
def test_tree_attention_refusals(lib, change, rc, text):
    from fused_turboquant_b200 import _lib
    signs, levels = np.ones(128, np.float32), np.linspace(-2, 2, 16).astype(np.float32)
    need = lib.ftq_tree_workspace_bytes(2, 8, 8, 2, 128, 64)
    assert need > 0
    good = dict(q=A, q_dtype=_lib.BF16, out=A, out_dtype=_lib.BF16, pool=A, num_blocks=8, block_table=A, max_blocks=4, seq_lens=A,
                max_seq_len=64, tree_lens=None, masks=A, B=2, n_nodes=8, Hq=8, Hkv=2, head_dim=128, bits_k=4, bits_v=4,
                levels_k=_lib.fptr(levels), levels_v=_lib.fptr(levels), signs=_lib.fptr(signs), scale=0.1, workspace=A,
                workspace_bytes=need, stream=None)
    assert _lib.F32 == 0
    got, message = call(lib, "ftq_tree_attn", good, **change)
    assert got == rc and text in message, (got, message)


def test_empty_calls_do_nothing(lib):
    assert call(lib, "ftq_pages_extend", EXTEND, n_requests=0)[0] == 0
    assert call(lib, "ftq_pages_trim", TRIM, n_requests=0)[0] == 0
    assert call(lib, "ftq_tree_masks", MASKS, B=0)[0] == 0
    assert call(lib, "ftq_tree_commit", COMMIT, B=0)[0] == 0
    assert call(lib, "ftq_logits_process", LOGITS, n_requests=0)[0] == 0
    assert call(lib, "ftq_logits_process", LOGITS, rows=0)[0] == 0


def test_workspace_sizes(lib):
    assert lib.ftq_logits_workspace_bytes(0, 100) >= 0
    # 8 bytes a row and segment of the vocabulary
    assert lib.ftq_logits_workspace_bytes(10, 131072) >= 10 * 8
    assert lib.ftq_tree_workspace_bytes(2, 0, 8, 2, 128, 64) == 0
    assert lib.ftq_tree_workspace_bytes(2, 257, 8, 2, 128, 64) == 0
    assert lib.ftq_tree_workspace_bytes(2, 8, 8, 3, 128, 64) == 0
    a, b = (lib.ftq_tree_workspace_bytes(n, 8, 32, 8, 128, 4096) for n in (1, 64))
    assert 0 < a < b


@pytest.mark.parametrize("out", ["path", "n_accepted", "out_tokens", "new_lens"])
@pytest.mark.parametrize("read", ["seq_lens", "tree_lens", "tokens", "parents", "next_tokens", "block_table"])
def test_what_a_commit_writes_lies_apart_from_what_it_reads(lib, out, read):
    """Every output on every input, from the first byte on and at its last; the rest of the call is sound."""
    size = dict(seq_lens=8, tree_lens=8, tokens=64, parents=64, next_tokens=64, block_table=32, path=64, n_accepted=8, out_tokens=64, new_lens=8)
    good = dict(COMMIT, tree_lens=1, **{})
    for i, name in enumerate(size):
        good[name] = (A << 4) + 4096 * i
    for at in (0, size[read] - 4, 4 - size[out]):
        rc, message = call(lib, "ftq_tree_commit", dict(good, **{out: good[read] + at}))
        assert rc == INVALID and "memory of their own" in message
