"""Prefill over keys that mask with the type's lowest value, whose scores are finite: they weigh nothing beside others."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_paged_serving import relative  # noqa: E402
from test_paged_serving_paths import LOWEST  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["split", "bf16"])
@pytest.mark.parametrize("scale", [128 ** -0.5, 0.125])
@pytest.mark.parametrize("size", [2.0 ** -6, 0.5, 1.0, 8.0])  # 8: the scores are -inf
@pytest.mark.parametrize("where", ["first", "middle", "last", "most"])
def test_prefill_of_keys_that_mask(monkeypatch, precision, scale, size, where):
    from lara_b200 import ops
    from lara_b200._native import lib

    monkeypatch.setenv("LARA_TC_SPLIT_P", "1" if precision == "split" else "0")
    B, hq, hkv, d, n, rows = 2, 4, 2, 128, 270, 800
    g = torch.Generator().manual_seed(int(size * 64))
    k, v = (torch.randn((B, hkv, rows, d), generator=g).bfloat16() for _ in "kv")
    q = torch.randn((B, n, hq, d), generator=g).bfloat16()
    q[..., :2] = size
    tokens = torch.tensor({"first": range(192), "middle": range(200, 400), "last": range(520, 660),
                           "most": range(513)}[where])
    k[:, :, tokens, :2] = LOWEST
    lens = torch.tensor([rows - n, 515], dtype=torch.int32)
    ws = ops.new_workspace(lib.lara_prefill_workspace_bytes(B, n, hq, hkv, d, rows), "cuda")
    got = ops.gqa_prefill(q.cuda(), k.cuda(), v.cuda(), lens.cuda(), scale=scale, workspace=ws)
    kd = k.double()
    kd[:, :, tokens] = 0.0
    kd, vd = (x.repeat_interleave(hq // hkv, 1) for x in (kd, v.double()))
    qd = q.double().transpose(1, 2)
    s = qd @ kd.transpose(2, 3) * scale
    hidden = torch.arange(rows) > lens.view(B, 1, 1, 1) + torch.arange(n).view(n, 1)
    hidden = hidden | torch.zeros(rows, dtype=torch.bool).index_fill_(0, tokens, True)
    p = torch.softmax(s.masked_fill(hidden, -float("inf")), -1)
    o, kappa = ((p @ x).transpose(1, 2) for x in (vd, vd.abs()))
    A = ((qd.abs() @ kd.abs().transpose(2, 3)) * scale).amax(-1, keepdim=True).transpose(1, 2)
    # The output's words are cut, not rounded: the reference's packer adds its carry below bit 16 (sw/attn_driver.py:88-98),
    # where the mask drops it.  A cut is off by less than one step, 2^-7 of the value, where a rounding is by half of one.
    tol = 2.0 ** -7 * o.abs() + kappa * relative(A, d, rows)
    if precision == "bf16":  # the weights are rounded once more
        tol += 2.0 ** -8 * kappa
    got = got.cpu().double()
    assert torch.isfinite(got).all() and ((got - o).abs() <= tol).all()
    assert ops.workspace_status(ws) == 0
