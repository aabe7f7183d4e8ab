"""A wait of the tree kernel that runs out, on purpose: rows become NaN, the status word says so, the next call is clean.

In `libftq_b200_waittest.so` the first half of CTA 0 never reports the scores of its second tile, and a wait ends after 4096 polls.
Nothing faults, traps or spins without bound.
"""
import ctypes
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [8, 40])    # two halves a CTA; one
def test_an_expired_wait_poisons_its_rows_and_nothing_else(t):
    import torch
    from fused_turboquant_b200 import PagedKVPool, _lib, build
    if not os.path.exists(build.TEST_LIB_PATH):
        pytest.skip("libftq_b200_waittest.so has not been built")
    bad_lib, good_lib = ctypes.CDLL(build.TEST_LIB_PATH), _lib.load()
    for name, (res, args) in _lib.SIGNATURES.items():
        fn = getattr(bad_lib, name)
        fn.restype, fn.argtypes = res, args
    # many long sequences: a share is several tiles, and no unit has more than a few shares
    d, hkv, group, B, n = 128, 8, 4, 16, 4096
    per = n // 16
    g = torch.Generator("cuda").manual_seed(4)
    table = torch.randperm(B * per, device="cuda", generator=g).int().view(B, per)
    pool = PagedKVPool(B * per, hkv, d, 4, 4)
    kv = torch.randn(2, B * n, hkv, d, device="cuda", generator=g).bfloat16()
    pool.store(kv[0], kv[1], torch.arange(B * n, device="cuda"), layer=0)
    q = torch.randn(B, t, hkv * group, d, device="cuda", generator=g).bfloat16()
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    words = (t + 31) // 32
    masks = torch.full((B, t, words), -1, dtype=torch.int32, device="cuda")
    ws = torch.empty(good_lib.ftq_tree_workspace_bytes(B, t, hkv * group, hkv, d, n), dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda x: ctypes.c_void_p(x.data_ptr())

    def run(lib):
        out = torch.full(q.shape, 7.0, device="cuda")
        rc = lib.ftq_tree_attn(p(q), _lib.BF16, p(out), _lib.F32, p(pool.pool[0]), pool.num_blocks, p(table), per, p(lens), n, None,
                               p(masks), B, t, hkv * group, hkv, d, 4, 4, _lib.fptr(pool.levels_k), _lib.fptr(pool.levels_v),
                               _lib.fptr(pool.signs), d ** -0.5, p(ws), ws.numel(), stream)
        assert rc == 0, lib.ftq_last_error()
        status = ctypes.c_int(-1)
        rc = lib.ftq_paged_decode_status(p(ws), 1, hkv * group, hkv, d, n, 1, stream, ctypes.byref(status))
        return out, rc, status.value

    good, rc, status = run(good_lib)
    assert rc == 0 and status == 0 and torch.isfinite(good).all()
    got, rc, status = run(bad_lib)
    assert rc == -5 and status == 2, (rc, status)
    heads = got.view(B, t, hkv, group * d)
    lost = torch.isnan(heads).any(-1)                       # [B, t, hkv]
    # all rows of a unit or none; the share of the first half of the first CTA and no other
    assert (lost == lost[:, :1]).all() if t * group <= 128 else True
    units = lost.any(1)
    assert units.any() and units[0, 0] and units.sum() <= 3 and not units[1:].any()
    keep = ~lost[..., None].expand_as(heads)
    assert torch.equal(heads[keep], good.view_as(heads)[keep])
    assert torch.isnan(heads[lost]).all()
    again, rc, status = run(good_lib)
    assert rc == 0 and status == 0 and torch.equal(again, good)


@pytest.mark.parametrize("t,rows", [(3, 16), (8, 32), (16, 64), (40, 128), (100, 128)])
def test_a_row_tile_is_lost_as_a_whole(t, rows):
    """Rows of node x head in tiles of `rows`: those of a tile belong to the same shares."""
    import torch
    from fused_turboquant_b200 import PagedKVPool, _lib, build
    if not os.path.exists(build.TEST_LIB_PATH):
        pytest.skip("libftq_b200_waittest.so has not been built")
    bad_lib, good_lib = ctypes.CDLL(build.TEST_LIB_PATH), _lib.load()
    for name, (res, args) in _lib.SIGNATURES.items():
        fn = getattr(bad_lib, name)
        fn.restype, fn.argtypes = res, args
    d, hkv, group, B, n = 128, 4, 4, 24, 3000
    per = -(-n // 16)
    g = torch.Generator("cuda").manual_seed(t)
    table = torch.randperm(B * per, device="cuda", generator=g).int().view(B, per)
    pool = PagedKVPool(B * per, hkv, d, 4, 4)
    kv = torch.randn(2, B * per * 16, hkv, d, device="cuda", generator=g).bfloat16()
    pool.store(kv[0], kv[1], torch.arange(B * per * 16, device="cuda"), layer=0)
    q = torch.randn(B, t, hkv * group, d, device="cuda", generator=g).bfloat16()
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    masks = torch.full((B, t, (t + 31) // 32), -1, dtype=torch.int32, device="cuda")
    ws = torch.empty(good_lib.ftq_tree_workspace_bytes(B, t, hkv * group, hkv, d, n), dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda x: ctypes.c_void_p(x.data_ptr())

    def run(lib):
        out = torch.full(q.shape, 7.0, device="cuda")
        rc = lib.ftq_tree_attn(p(q), _lib.BF16, p(out), _lib.F32, p(pool.pool[0]), pool.num_blocks, p(table), per, p(lens), n, None,
                               p(masks), B, t, hkv * group, hkv, d, 4, 4, _lib.fptr(pool.levels_k), _lib.fptr(pool.levels_v),
                               _lib.fptr(pool.signs), d ** -0.5, p(ws), ws.numel(), stream)
        assert rc == 0, lib.ftq_last_error()
        status = ctypes.c_int(-1)
        lib.ftq_paged_decode_status(p(ws), 1, hkv * group, hkv, d, n, 1, stream, ctypes.byref(status))
        return out, status.value

    for _ in range(2):
        good, status = run(good_lib)
        assert status == 0 and torch.isfinite(good).all()
        got, status = run(bad_lib)
        assert status == 2
        by_row = lambda x: x.view(B, t, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(B, hkv, t * group, d)  # noqa: E731
        nan = by_row(got).isnan()
        lost = nan.any(-1)
        assert torch.equal(lost, nan.all(-1))
        tiles = 0
        for r in range(0, t * group, rows):
            part = lost[:, :, r:r + rows]
            assert torch.equal(part.any(-1), part.all(-1)) and not part[1:].any()
            tiles += int(part.all(-1).sum())
        assert 1 <= tiles <= 3
        assert torch.equal(by_row(got)[~lost], by_row(good)[~lost])
