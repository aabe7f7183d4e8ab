"""The wait of shared attention for its queries that runs out, on purpose: rows become NaN, the status word says so, the next call is
clean.

In `libftq_b200_waittest.so` warp 5 of CTA 0 announces the queries of its first piece to their mbarrier but does not ask for them where a
group has five rows, and a wait ends after 64 polls.  Nothing faults, traps or spins without bound.
"""
import ctypes
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K,group,d", [(5, 1, 128), (5, 3, 128), (5, 6, 128)])    # one, two and four tiles of columns
def test_queries_that_never_come_poison_their_rows_and_nothing_else(K, group, d):
    import torch
    from fused_turboquant_b200 import PagedKVPool, _lib, build
    if not os.path.exists(build.TEST_LIB_PATH):
        pytest.skip("libftq_b200_waittest.so has not been built")
    bad_lib, good_lib = ctypes.CDLL(build.TEST_LIB_PATH), _lib.load()
    for name, (res, args) in _lib.SIGNATURES.items():
        fn = getattr(bad_lib, name)
        fn.restype, fn.argtypes = res, args
    # every warp has pages of a group's unit
    hkv, R, ctx, own = 8, 16, 4096, 40
    n, per = ctx + own, 259
    g = torch.Generator("cuda").manual_seed(4)
    blocks = R * (256 + 3 * K)
    ids = torch.randperm(blocks, device="cuda", generator=g).int()
    table = torch.cat([ids[:R * 256].view(R, 1, 256).expand(R, K, 256), ids[R * 256:].view(R, K, 3)], -1).reshape(R * K, per).contiguous()
    pool = PagedKVPool(blocks, hkv, d, 4, 4)
    kv = torch.randn(2, blocks * 16, hkv, d, device="cuda", generator=g).bfloat16()
    pool.store(kv[0], kv[1], torch.arange(blocks * 16, device="cuda"), layer=0)
    q = torch.randn(R * K, hkv * group, d, device="cuda", generator=g).bfloat16()
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, shared = torch.full((R * K,), n, **i32), torch.full((R,), ctx, **i32)
    ws = torch.empty(good_lib.ftq_shared_workspace_bytes(R, K, hkv * group, hkv, d, n), dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda x: ctypes.c_void_p(x.data_ptr())   # noqa: E731

    def run(lib):
        out = torch.full(q.shape, 7.0, device="cuda")
        rc = lib.ftq_shared_attn(p(q), _lib.BF16, p(out), _lib.F32, p(pool.pool[0]), pool.num_blocks, p(table), per, p(lens), n, p(shared), R, K,
                                 hkv * group, hkv, d, 4, 4, _lib.fptr(pool.levels_k), _lib.fptr(pool.levels_v), _lib.fptr(pool.signs), d ** -0.5,
                                 p(ws), ws.numel(), stream)
        assert rc == 0, lib.ftq_last_error()
        status = ctypes.c_int(-1)
        rc = lib.ftq_paged_decode_status(p(ws), 1, hkv * group, hkv, d, n, 1, stream, ctypes.byref(status))
        return out, rc, status.value

    good, rc, status = run(good_lib)
    assert rc == 0 and status == 0 and torch.isfinite(good).all()
    got, rc, status = run(bad_lib)
    assert rc == -5 and status == 2, (rc, status)
    heads = got.view(R, K, hkv, group * d)
    nan = torch.isnan(heads)
    lost = nan.any(-1)                                  # [R, K, hkv]
    assert torch.equal(lost, nan.all(-1))
    # whole units of a group (a warp's share: one or two of them) and the rows that the warp has besides
    units = lost.all(1)
    assert 1 <= int(units.sum()) <= 2 and 0 <= int(lost.sum()) - K * int(units.sum()) <= 8
    assert torch.equal(heads[~lost], good.view_as(heads)[~lost])
    again, rc, status = run(good_lib)
    assert rc == 0 and status == 0 and torch.equal(again, good)
