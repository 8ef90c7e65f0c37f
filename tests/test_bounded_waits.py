"""Kernels whose waits run out end, report it, and leave the GPU usable; nothing here faults or hangs one."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_paged_serving import check_out, decode64, dev, make_cache  # noqa: E402


@pytest.fixture
def withhold():
    """Loads that bring some tiles and then no more."""
    from lara_b200._native import lib

    yield lib.lara_selftest_withhold_tiles
    lib.lara_selftest_withhold_tiles(-1)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,batch,page,shared", [
    (16, 8, 128, 3, 64, 300),     # one row tile; CTAs that have parts of two kv heads
    (16, 8, 64, 80, 64, 400),     # pairs of row tiles
    (16, 16, 64, 1500, 16, 16)])  # and CTAs with many short units each
@pytest.mark.parametrize("brought", [0, 1, 4])
def test_shared_decode_whose_waits_run_out(withhold, hq, hkv, d, batch, page, shared, brought):
    """A workspace of which nothing makes sense at first: what a call reads of it, it has written, also when it fails."""
    from lara_b200 import ops, paged

    k, v, table, n = make_cache([shared * page + 5] * batch, hkv, d, page, seed=3, shared=shared)
    q = torch.randn((batch, hq, d), generator=torch.Generator().manual_seed(1)).bfloat16()
    qd, kd, vd, td, nd = dev(q, k, v, table, n)
    ws = paged.shared_workspace(batch, hq, hkv, d, "cuda")
    ws[256:] = 0x7f
    withhold(brought)
    paged.gqa_decode_shared(qd, kd, vd, td, nd, shared, workspace=ws)
    withhold(-1)
    assert ops.workspace_status(ws) == 1  # a wait ran out
    o, kappa, A, _ = decode64(qd, kd, vd, td, nd, page, d ** -0.5)
    check_out(paged.gqa_decode_shared(qd, kd, vd, td, nd, shared, workspace=ws), o, kappa, A, n)
    assert ops.workspace_status(ws) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["split", "bf16"])
@pytest.mark.parametrize("brought", [0, 1, 3])
def test_prefill_whose_waits_run_out(withhold, monkeypatch, precision, brought):
    from lara_b200 import ops
    from lara_b200._native import lib

    if precision == "bf16":
        monkeypatch.setenv("LARA_TC_SPLIT_P", "0")
    hq, hkv, d, n, rows = 4, 2, 128, 300, 900
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((2, hkv, rows, d), generator=g).bfloat16().cuda() for _ in "kv")
    q = torch.randn((2, n, hq, d), generator=g).bfloat16().cuda()
    lens = torch.tensor([rows - n, 290], dtype=torch.int32, device="cuda")
    ws = ops.new_workspace(lib.lara_prefill_workspace_bytes(2, n, hq, hkv, d, rows), "cuda")
    want = ops.gqa_prefill(q, k, v, lens, workspace=ws)
    assert ops.workspace_status(ws) == 0
    withhold(brought)
    ops.gqa_prefill(q, k, v, lens, workspace=ws)
    withhold(-1)
    assert ops.workspace_status(ws) == 1  # a wait ran out
    assert torch.equal(ops.gqa_prefill(q, k, v, lens, workspace=ws).view(torch.int16), want.view(torch.int16))
    assert ops.workspace_status(ws) == 0
