"""What attention with common blocks refuses besides, before anything is launched (no GPU)."""
import numpy as np
import pytest

A = 0x10000        # an address that nothing follows


@pytest.mark.parametrize("change,rc,text", [
    (dict(num_blocks=0), -1, "no blocks"),
    (dict(max_seq_len=1 << 30, max_blocks=1 << 26, n_requests=1, group=1024), -2, "too many tokens"),
])
def test_refusals(change, rc, text):
    from fused_turboquant_b200 import _lib, build
    build.build()
    lib = _lib.load()
    signs, levels = np.ones(128, np.float32), np.linspace(-2, 2, 16).astype(np.float32)
    good = dict(q=A, q_dtype=_lib.BF16, out=A, out_dtype=_lib.BF16, pool=A, num_blocks=8, block_table=A, max_blocks=4, seq_lens=A,
                max_seq_len=64, shared_lens=A, n_requests=2, group=4, Hq=8, Hkv=2, head_dim=128, bits_k=4, bits_v=4,
                levels_k=_lib.fptr(levels), levels_v=_lib.fptr(levels), signs=_lib.fptr(signs), scale=0.1, workspace=A,
                workspace_bytes=1 << 40, stream=None)
    got = lib.ftq_shared_attn(*{**good, **change}.values())
    assert got == rc and text in lib.ftq_last_error().decode()
