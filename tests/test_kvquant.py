"""8-bit KV cache (``lara_b200.kvquant``) and the q/k head pass (``ops.qk_norm_rope``).

Every operator is compared with its definition in 64 bits.  Tolerances:

* codes, scales and read-back values are exact (the definition says how each is
  rounded, and the roundings are reproducible);
* ``qk_norm_rope``: one bf16 rounding (2^-8 of the value: 8 significant bits) plus fp32 rounding of at
  most 16 steps of 2^-24 on each of the two terms of a rotated value;
* decode: one bf16 rounding (2^-8), plus, relative to ``kappa = sum_t p_t |v_t|``: weights
  held in fp16 (2^-11), scores in fp32 (136 roundings of 2^-24 of
  ``sum_d |q_d k_d|``, twice: in the sums above and below the line), sums in fp32
  over n tokens (n 2^-23), and weights too small for fp16 (n 2^-24 of the row's
  largest kappa).
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

FORMATS = ["int8", "fp8_e4m3"]
DTYPES = {"int8": torch.int8, "fp8_e4m3": torch.float8_e4m3fn}


# ------------------------------------------------------------------ definitions in 64 bits (CPU)
def quantise64(x: torch.Tensor, fmt: str):
    """rows [..., D] -> (code values [..., D], scales [...]) in float64."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(x).all(-1, keepdim=True)
    if fmt == "int8":
        a = a.clamp_min(2.0 ** -100)
        scale = a / 127.0
        codes = torch.round(127.0 * x / a)
    else:
        _, e = torch.frexp(a / 448.0)  # a / 448 = m 2^e, m in [0.5, 1)
        exact_power = torch.ldexp(torch.ones_like(a), e - 1) == a / 448.0
        e = torch.where(exact_power, e - 1, e).clamp_min(-100)
        e = torch.where(a == 0, torch.full_like(e, -100), e)
        scale = torch.ldexp(torch.ones_like(a), e)
        y = x / scale
        _, ye = torch.frexp(y.abs().clamp_min(2.0 ** -6))
        step = torch.ldexp(torch.ones_like(y), ye - 4)
        codes = torch.round(y / step) * step
    codes = torch.where(ok, codes, torch.zeros_like(codes))
    return codes, torch.where(ok, scale, torch.full_like(scale, math.nan)).squeeze(-1)


def values64(codes, scales):
    return codes * scales[..., None]


def norm_rope64(x, w, cos, sin, interleaved, eps):
    """x [..., H, D] float64 -> (result, the bound's magnitude of the two terms)."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    out, mag = y.clone(), y.abs()
    if cos is not None:
        half = cos.shape[-1]
        i = torch.arange(half)
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
        a, b = y[..., ia], y[..., ib]
        out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
        mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return out, mag


def attend64(q, k, v, scale):
    """q [G, D], k/v [n, D] float64 -> (o [G, D], absolute tolerance [G, D])."""
    n = k.shape[0]
    s = (q @ k.T) * scale
    mag = (q.abs() @ k.abs().T) * scale
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o, kappa = p @ v, p @ v.abs()
    err_s = 136 * 2.0 ** -24 * (p * mag).sum(-1, keepdim=True).maximum(mag.amax(-1, keepdim=True) * 2.0 ** -3)
    rel = 2.0 ** -11 + 2 * err_s + n * 2.0 ** -23 + 2.0 ** -20
    tol = 2.0 ** -8 * o.abs() + rel * kappa + n * 2.0 ** -24 * kappa.amax(-1, keepdim=True)
    return o, tol + 2.0 ** -133


# ------------------------------------------------------------------ CPU tests
def _lib():
    from lara_b200 import _native

    return _native


def _pool_struct(**kw):
    n = _lib()
    d = dict(k_codes=4096, v_codes=4096, k_scales=4096, v_scales=4096, format=0, num_pages=4, n_kv_heads=2,
             page_size=64, head_dim=128)
    d.update(kw)
    return n.LaraKvqPool(*[d[f] for f, _ in n.LaraKvqPool._fields_])


P = ctypes.c_void_p(4096)


def _append(pool, table=P, pps=4, starts=P, counts=None, new_lens=None, k=P, v=P, batch=1, n=1):
    return _lib().lib.lara_kvq_append(ctypes.byref(pool), table, pps, starts, counts, new_lens, k, 0, 0, 0, v, 0, 0, 0,
                                      batch, n, None, None)


def _read(pool, lens=P, k=P, batch=1, n=1, pps=4):
    return _lib().lib.lara_kvq_read(ctypes.byref(pool), P, pps, lens, None, k, 0, 0, 0, P, 0, 0, 0, batch, n, None,
                                    None)


def _decode(pool, q=P, batch=1, hq=8, scale=0.1, ws=P, wsb=1 << 30, pps=4, lens=P):
    return _lib().lib.lara_gqa_decode_kvq(q, ctypes.byref(pool), P, pps, lens, P, batch, hq, scale, ws, wsb, None)


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=96), 0x22), (dict(format=2), 0x22), (dict(page_size=48), 0x01), (dict(page_size=8), 0x01),
    (dict(page_size=1 << 17), 0x01), (dict(num_pages=0), 0x01), (dict(n_kv_heads=0), 0x01),
    (dict(k_codes=None), 0x11), (dict(v_scales=None), 0x11), (dict(v_codes=4100), 0x11), (dict(k_scales=4100), 0x11)])
def test_bad_pools_are_refused_by_every_call(kw, code):
    pool = _pool_struct(**kw)
    assert _append(pool) == code
    assert _read(pool) == code
    assert _decode(pool) == code


def test_refusals_before_any_launch():
    pool = _pool_struct()
    assert _append(pool, table=None) == 0x11
    assert _append(pool, starts=None) == 0x11
    assert _append(pool, k=None) == 0x11
    assert _append(pool, k=ctypes.c_void_p(4097)) == 0x11
    assert _append(pool, new_lens=P) == 0x11  # aliases starts
    assert _append(pool, batch=-1) == 0x01
    assert _append(pool, n=-1) == 0x01
    assert _append(pool, pps=0) == 0x01
    assert _append(pool, pps=1 << 26) == 0x01  # capacity past int32
    assert _append(pool, batch=65535, n=1 << 20) == 0x01
    assert _read(pool, lens=None) == 0x11
    assert _read(pool, k=None) == 0x11
    assert _read(pool, n=-1) == 0x01
    assert _decode(pool, hq=7) == 0x01
    assert _decode(pool, hq=34) == 0x22  # 17 heads per kv head
    assert _decode(pool, scale=0.0) == 0x01
    assert _decode(pool, scale=math.inf) == 0x01
    assert _decode(pool, scale=math.nan) == 0x01
    assert _decode(pool, q=None) == 0x11
    assert _decode(pool, q=ctypes.c_void_p(4104)) == 0x11
    assert _decode(pool, ws=None) == 0x11
    assert _decode(pool, wsb=16) == 0x12
    assert _decode(pool, batch=70000) == 0x01
    # nothing to do is not an error
    assert _append(pool, batch=0) == 0
    assert _append(pool, n=0, k=None, v=None) == 0
    assert _read(pool, n=0) == 0
    assert _decode(pool, batch=0) == 0
    assert _lib().lib.lara_kvq_decode_workspace_bytes(0, 8, 2, 128) == 0


def _norm_rope(q=P, hd=128, n=1, hq=8, hkv=2, pos=P, table=P, max_pos=16, rot=128, qw=P, kw=P, eps=1e-5):
    z = (0, 0, 0)
    return _lib().lib.lara_qk_norm_rope(q, *z, P, *z, P, *z, P, *z, 1, n, hq, hkv, hd, pos, table, max_pos, rot, 1, qw,
                                        kw, eps, None, None)


def _append_qkv(pool, q=P, v=P, starts=P, new_lens=None, batch=1, n=1, hq=8, table=P, rot=128, qw=P, kw=P, eps=1e-5):
    z = (0, 0, 0)
    return _lib().lib.lara_kvq_append_qkv(ctypes.byref(pool), P, 4, starts, None, new_lens, q, *z, P, *z, v, *z, P, *z,
                                          batch, n, hq, None, table, 16, rot, 1, qw, kw, eps, None, None)


def test_append_qkv_refusals():
    pool = _pool_struct()
    assert _append_qkv(_pool_struct(head_dim=80)) == 0x22
    assert _append_qkv(pool, rot=12) == 0x01
    assert _append_qkv(pool, hq=0) == 0x01
    assert _append_qkv(pool, n=-1) == 0x01
    assert _append_qkv(pool, batch=1 << 20, n=1 << 10) == 0x01
    assert _append_qkv(pool, kw=None) == 0x01
    assert _append_qkv(pool, eps=-1.0) == 0x01
    assert _append_qkv(pool, q=None) == 0x11
    assert _append_qkv(pool, v=None) == 0x11
    assert _append_qkv(pool, starts=None) == 0x11
    assert _append_qkv(pool, new_lens=P) == 0x11
    assert _append_qkv(pool, qw=ctypes.c_void_p(4104)) == 0x11
    assert _append_qkv(pool, batch=0) == 0
    assert _append_qkv(pool, n=0, q=None, v=None) == 0


def test_norm_rope_refusals():
    assert _norm_rope(hd=96) == 0x22
    assert _norm_rope(hq=0) == 0x01
    assert _norm_rope(rot=4) == 0x01
    assert _norm_rope(rot=136) == 0x01
    assert _norm_rope(max_pos=0) == 0x01
    assert _norm_rope(qw=None) == 0x01  # one weight without the other
    assert _norm_rope(qw=None, kw=None, table=None) == 0x01  # nothing to do
    assert _norm_rope(eps=-1.0) == 0x01
    assert _norm_rope(eps=math.nan) == 0x01
    assert _norm_rope(q=None) == 0x11
    assert _norm_rope(pos=None) == 0x11
    assert _norm_rope(table=ctypes.c_void_p(4104)) == 0x11
    assert _norm_rope(n=0, q=None) == 0


def test_python_checks():
    from lara_b200 import kvquant, ops

    c = torch.zeros((4, 2, 16, 64), dtype=torch.int8)
    s = torch.zeros((4, 2, 16))
    with pytest.raises(ValueError, match="CUDA"):
        kvquant.QuantPool(c, c, s, s)
    with pytest.raises(TypeError, match="int8"):
        kvquant.QuantPool(c.float(), c, s, s)
    with pytest.raises(ValueError, match="fmt"):
        kvquant.QuantPool.empty(4, 16, 2, 64, fmt="int3", device="cpu")
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.rope_table(16, 12, device="cpu")
    x = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.qk_norm_rope(x, x)
    with pytest.raises(TypeError, match="bf16"):
        ops.qk_norm_rope(x.float(), x)


def test_rope_table_matches_the_angles():
    from lara_b200 import ops

    t = ops.rope_table(1000, 64, base=500000.0, device="cpu").double()
    pos, i = np.arange(1000)[:, None], np.arange(32)[None]
    ang = pos * 500000.0 ** (-2.0 * i / 64)
    assert np.abs(t[:, :32].numpy() - np.cos(ang)).max() <= 2.0 ** -25 + 1e-12
    assert np.abs(t[:, 32:].numpy() - np.sin(ang)).max() <= 2.0 ** -25 + 1e-12


# ------------------------------------------------------------------ GPU helpers
DEV = "cuda:0"


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")


def _rand_bf16(g, shape, outliers=True):
    x = torch.randn(shape, generator=g)
    if outliers:
        x[..., 3] *= 12.0
    return x.to(torch.bfloat16)


def _table(g, lens, pps, ps, extra=0):
    """Block table over randomly ordered pages; entries past a sequence's last page are -1."""
    used = [-(-n // ps) for n in lens]
    perm = torch.randperm(sum(used) + extra, generator=g).to(torch.int32)
    t = torch.full((len(lens), pps), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        t[b, :u] = perm[at:at + u]
        at += u
    return t, max(1, sum(used) + extra)


class Case:
    """A pool of garbage with the given sequences quantised into it on the CPU, by the definition."""

    def __init__(self, lens, hkv, D, ps, fmt, seed=0, capacity=None, k_rows=None, v_rows=None):
        from lara_b200 import kvquant

        _need_gpu()
        g = torch.Generator().manual_seed(seed)
        self.lens, self.fmt, self.D, self.hkv, self.ps = list(lens), fmt, D, hkv, ps
        cap = max(max(lens), 1) if capacity is None else capacity
        self.table, pages = _table(g, lens, -(-cap // ps), ps, extra=2)
        # every byte pattern (e4m3's NaN codes too) and scales of NaN, infinity and zero outside the valid rows
        raw = [torch.randint(0, 256, (pages, hkv, ps, D), generator=g).to(torch.uint8) for _ in range(2)]
        bad = torch.tensor([math.nan, math.inf, -math.inf, 0.0, 1e30])
        sc = [bad[torch.randint(0, 5, (pages, hkv, ps), generator=g)] for _ in range(2)]
        self.k64, self.v64 = [], []
        for b, n in enumerate(lens):
            rows = [r[b] if r is not None else _rand_bf16(g, (hkv, n, D)) for r in (k_rows, v_rows)]
            for x, codes, scales, keep in zip(rows, raw, sc, (self.k64, self.v64)):
                c, s = quantise64(x, fmt)
                keep.append(values64(c, s.float().double()))
                bits = (c.to(torch.int8) if fmt == "int8" else c.float().to(torch.float8_e4m3fn)).view(torch.uint8)
                for t in range(n):
                    p = int(self.table[b, t // ps])
                    codes[p, :, t % ps] = bits[:, t]
                    scales[p, :, t % ps] = s[:, t].float()
        dt = DTYPES[fmt]
        self.pool = kvquant.QuantPool(*[r.to(DEV).view(dt) for r in raw], *[s.to(DEV) for s in sc])
        self.dtable = self.table.to(DEV)
        self.dlens = torch.tensor(self.lens, dtype=torch.int32, device=DEV)

    def check(self, q, o, scale=None):
        """o[B, Hq, D] against attention in 64 bits."""
        sc = 1.0 / math.sqrt(self.D) if scale is None else scale
        G = q.shape[1] // self.hkv
        o = o.double().cpu()
        for b, n in enumerate(self.lens):
            for h in range(self.hkv):
                got = o[b, h * G:(h + 1) * G]
                if n == 0:
                    assert torch.count_nonzero(got) == 0
                    continue
                ref, tol = attend64(q[b, h * G:(h + 1) * G].double().cpu(), self.k64[b][h], self.v64[b][h], sc)
                bad = (got - ref).abs() > tol
                assert not bad.any(), (b, h, n, (got - ref).abs().max(), ((got - ref).abs() / tol).max())


def _decode_gpu(case, q, **kw):
    from lara_b200 import kvquant, ops

    B, hq, D = q.shape
    ws = kvquant.decode_workspace(B, hq, case.hkv, D, DEV)
    o = kvquant.gqa_decode_kvq(q, case.pool, case.dtable, case.dlens, workspace=ws, **kw)
    assert ops.workspace_status(ws) == 0
    return o


# ------------------------------------------------------------------ qk_norm_rope
@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 7, 129])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 64), (64, 8)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (5, 1)])
def test_norm_rope(T, D, rot, interleaved, hq, hkv):
    _need_gpu()
    from lara_b200 import ops

    g = torch.Generator().manual_seed(T + D + rot + hq)
    q, k = _rand_bf16(g, (T, hq, D)), _rand_bf16(g, (T, hkv, D))
    q[0, 0] = 0.0  # a head of zeros: eps alone under the root
    qw, kw = (_rand_bf16(g, (D,), False) for _ in range(2))
    pos = torch.randint(0, 70000, (T,), generator=g).to(torch.int32)
    pos[0] = 69999
    tab = ops.rope_table(70000, rot, device="cpu")
    cs = tab[pos.long()]
    dtab = tab.to(DEV)
    for norm, rope in ((True, True), (False, True), (True, False)):
        st = ops.new_workspace(256, DEV)
        got = ops.qk_norm_rope(q.to(DEV), k.to(DEV), positions=pos.to(DEV) if rope else None,
                               cos_sin=dtab if rope else None, q_weight=qw.to(DEV) if norm else None,
                               k_weight=kw.to(DEV) if norm else None, interleaved=interleaved, workspace=st)
        assert ops.workspace_status(st) == 0
        for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
            ref, mag = norm_rope64(x, w if norm else None, cs[:, :rot // 2] if rope else None, cs[:, rot // 2:],
                                   interleaved, float(np.float32(1e-5)))
            err = (y.double().cpu() - ref).abs()
            bad = err > 2.0 ** -8 * ref.abs() + 16 * 2.0 ** -24 * mag + 2.0 ** -133
            assert int(bad.sum()) == 0


@pytest.mark.gpu
def test_norm_rope_views_and_in_place():
    """Packed projections, head-major layouts, odd strides and in-place calls give the same words."""
    _need_gpu()
    from lara_b200 import ops

    g = torch.Generator().manual_seed(5)
    B, n, hq, hkv, D = 3, 11, 8, 2, 128
    x = _rand_bf16(g, (B, n, hq + 2 * hkv, D)).to(DEV)
    q, k = x[:, :, :hq], x[:, :, hq:hq + hkv]
    w = _rand_bf16(g, (2, D), False).to(DEV)
    pos = torch.randint(0, 500, (B, n), generator=g).to(torch.int32).to(DEV)
    kw = dict(positions=pos, cos_sin=ops.rope_table(500, D, device=DEV), q_weight=w[0], k_weight=w[1])
    ref = ops.qk_norm_rope(q.contiguous(), k.contiguous(), **kw)
    views = ops.qk_norm_rope(q, k, **kw)
    flat = dict(kw, positions=pos.flatten())
    three = ops.qk_norm_rope(q.reshape(B * n, hq, D), k.reshape(B * n, hkv, D), **flat)
    hm = [torch.empty((B, h, n, D), dtype=torch.bfloat16, device=DEV) for h in (hq, hkv)]
    ops.qk_norm_rope(q, k, **kw, out=tuple(t.transpose(1, 2) for t in hm))
    pad = torch.zeros((B, n, hq + hkv, D + 3), dtype=torch.bfloat16, device=DEV)  # rows at odd addresses
    pad[..., 1:D + 1] = x[:, :, :hq + hkv]
    odd = ops.qk_norm_rope(pad[:, :, :hq, 1:D + 1], pad[:, :, hq:, 1:D + 1], **kw)
    y = x.clone()
    ops.qk_norm_rope(y[:, :, :hq], y[:, :, hq:hq + hkv], **kw, out=(y[:, :, :hq], y[:, :, hq:hq + hkv]))
    assert torch.equal(y[:, :, hq + hkv:], x[:, :, hq + hkv:])
    for i in range(2):
        assert torch.equal(views[i], ref[i]) and torch.equal(odd[i], ref[i])
        assert torch.equal(three[i].view(ref[i].shape), ref[i])
        assert torch.equal(hm[i].transpose(1, 2), ref[i])
        assert torch.equal((y[:, :, :hq], y[:, :, hq:hq + hkv])[i], ref[i])


@pytest.mark.gpu
def test_norm_rope_bad_positions_and_nan():
    _need_gpu()
    from lara_b200 import ops

    g = torch.Generator().manual_seed(6)
    q, k = _rand_bf16(g, (4, 2, 64)).to(DEV), _rand_bf16(g, (4, 1, 64)).to(DEV)
    tab = ops.rope_table(10, 64, device=DEV)
    st = ops.new_workspace(256, DEV)
    bad = torch.tensor([3, -1, 10, 2 ** 30], dtype=torch.int32, device=DEV)
    near = torch.tensor([3, 0, 9, 9], dtype=torch.int32, device=DEV)
    got = ops.qk_norm_rope(q, k, positions=bad, cos_sin=tab, workspace=st)
    assert ops.workspace_status(st) == 0x10
    ref = ops.qk_norm_rope(q, k, positions=near, cos_sin=tab, workspace=st)
    assert ops.workspace_status(st) == 0
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    q2 = q.clone()
    q2[1, 0, 5] = math.nan
    a = ops.qk_norm_rope(q, k, positions=near, cos_sin=tab, q_weight=w, k_weight=w)
    b = ops.qk_norm_rope(q2, k, positions=near, cos_sin=tab, q_weight=w, k_weight=w)
    assert torch.isnan(b[0][1, 0]).all()  # the head's norm, and nothing else
    b[0][1, 0] = a[0][1, 0]
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------ append and read
def _edge_rows(g, n, D):
    """bf16 rows of every kind: ordinary, ties, zeros, subnormals, huge, NaN and infinite."""
    x = torch.randn((n, D), generator=g) * torch.exp2(torch.randint(-30, 30, (n, 1), generator=g).float())
    x = x.to(torch.bfloat16)
    kinds = [0.0, 1e-38, 2.0 ** -133, 3e38, 1.0, 224.0, 225.0, 448.0, 127.0, 254.0]
    for i, a in enumerate(kinds[:n]):
        x[i] = (torch.randint(-8, 9, (D,), generator=g).float() / 16.0 * a).to(torch.bfloat16)  # ties at a/2 and more
        x[i, 7] = a
    if n > 12:
        x[10, 3], x[11, D - 1], x[12, 0] = math.nan, math.inf, -math.inf
        x[13:14] = -0.0
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ps", [16, 64])
@pytest.mark.parametrize("layout", ["head_major", "token_major", "odd"])
def test_append_codes_and_read_back(fmt, D, ps, layout):
    _need_gpu()
    from lara_b200 import kvquant, ops

    g = torch.Generator().manual_seed(D + ps)
    starts, counts, n, hkv = [0, 5, ps - 1, 3 * ps, 17], [40, 0, 1, 33, 40], 40, 3
    lens = [s + c for s, c in zip(starts, counts)]
    table, pages = _table(g, lens, 8, ps, extra=3)
    B = len(starts)
    k, v = (_edge_rows(g, B * hkv * n, D).view(B, hkv, n, D) for _ in range(2))
    if layout == "head_major":
        kd, vd = k.to(DEV), v.to(DEV)
    elif layout == "token_major":
        kd, vd = (x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for x in (k, v))
    else:
        kd, vd = (torch.nn.functional.pad(x, (1, 2)).to(DEV)[..., 1:D + 1] for x in (k, v))
    pool = kvquant.QuantPool.empty(pages, ps, hkv, D, fmt, DEV)
    for t in (pool.k_codes, pool.v_codes):
        t.view(torch.int8).fill_(77)
    pool.k_scales.fill_(-5.0)
    pool.v_scales.fill_(-5.0)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    st, new = ops.new_workspace(256, DEV), i32([-9] * B)
    kvquant.kvq_append(pool, table.to(DEV), i32(starts), kd, vd, counts=i32(counts), new_lens=new, workspace=st)
    assert ops.workspace_status(st) == 0
    assert new.tolist() == lens
    ko, vo = kvquant.kvq_read(pool, table.to(DEV), new, n, starts=i32(starts), workspace=st)
    assert ops.workspace_status(st) == 0
    for x, codes, scales, back in ((k, pool.k_codes, pool.k_scales, ko), (v, pool.v_codes, pool.v_scales, vo)):
        c64, s64 = quantise64(x, fmt)
        bits = (c64.to(torch.int8) if fmt == "int8" else c64.float().to(torch.float8_e4m3fn)).view(torch.uint8)
        want_c = torch.full((pages, hkv, ps, D), 77, dtype=torch.uint8)
        want_s = torch.full((pages, hkv, ps), -5.0)
        want_v = torch.zeros((B, hkv, n, D))
        for b in range(B):
            for t in range(counts[b]):
                p, r = int(table[b, (starts[b] + t) // ps]), (starts[b] + t) % ps
                want_c[p, :, r], want_s[p, :, r] = bits[b, :, t], s64[b, :, t].float()
                want_v[b, :, t] = c64[b, :, t].float() * s64[b, :, t, None].float()
        got_c = codes.view(torch.uint8).cpu()
        if fmt == "fp8_e4m3":  # the sign of a zero is kept, but is not part of the value
            got_c, want_c = (torch.where(z == 0x80, torch.zeros_like(z), z) for z in (got_c, want_c))
        assert torch.equal(got_c, want_c)
        assert torch.equal(scales.cpu().nan_to_num(1e9), want_s.nan_to_num(1e9))
        want_v, back = want_v.to(torch.bfloat16), back.cpu()
        assert torch.equal(torch.isnan(back), torch.isnan(want_v))
        assert torch.equal(back.nan_to_num(0.0), want_v.nan_to_num(0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_append_overflow_bad_pages_and_counts(fmt):
    _need_gpu()
    from lara_b200 import kvquant, ops

    g = torch.Generator().manual_seed(1)
    hkv, D, ps, n = 2, 64, 16, 20
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    pool = kvquant.QuantPool.empty(6, ps, hkv, D, fmt, DEV)
    table = i32([[0, 1], [2, 3], [4, 99]])
    x = _rand_bf16(g, (3, hkv, n, D)).to(DEV)
    st, new = ops.new_workspace(256, DEV), i32([0] * 3)
    kvquant.kvq_append(pool, table, i32([20, 0, 0]), x, x, new_lens=new, workspace=st)
    assert ops.workspace_status(st) == 0x4 | 0x8  # sequence 0 overflows, sequence 2 names page 99
    assert new.tolist() == [32, 20, 20]
    k, _ = kvquant.kvq_read(pool, table, i32([32, 20, 20]), 32, workspace=st)
    assert ops.workspace_status(st) == 0x8
    c, s = quantise64(x.cpu(), fmt)
    want = (c.float() * s.float()[..., None]).to(torch.bfloat16)
    assert torch.equal(k[0, :, 20:].cpu(), want[0, :, :12]) and torch.count_nonzero(k[0, :, :20]) == 0
    assert torch.equal(k[1, :, :20].cpu(), want[1])
    assert torch.equal(k[2, :, :16].cpu(), want[2, :, :16]) and torch.count_nonzero(k[2, :, 16:]) == 0
    kvquant.kvq_append(pool, table[:1], i32([-3]), x[:1], x[:1], new_lens=new[:1], workspace=st)
    assert ops.workspace_status(st) == 0x4
    kvquant.kvq_append(pool, table[1:2], i32([0]), x[:1], x[:1], counts=i32([21]), workspace=st)
    assert ops.workspace_status(st) == 0x2  # clamped to n
    kvquant.kvq_read(pool, table[:1], i32([33]), 32, workspace=st)
    assert ops.workspace_status(st) == 0x2
    # no rows: only the lengths
    e = torch.empty((3, hkv, 0, D), dtype=torch.bfloat16, device=DEV)
    kvquant.kvq_append(pool, table, i32([7, 8, 9]), e, e, new_lens=new, workspace=st)
    assert new.tolist() == [7, 8, 9] and ops.workspace_status(st) == 0


@pytest.mark.gpu
def test_read_into_a_cache_slice_and_odd_strides():
    _need_gpu()
    from lara_b200 import kvquant

    case = Case([50, 0, 33], 2, 128, 16, "int8", seed=3)
    k, v = kvquant.kvq_read(case.pool, case.dtable, case.dlens, 50)
    big = torch.full((2, 3, 2, 64, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    kvquant.kvq_read(case.pool, case.dtable, case.dlens, 50, out=(big[0, :, :, :50], big[1, :, :, :50]))
    assert torch.equal(big[0, :, :, :50], k) and torch.equal(big[1, :, :, :50], v)
    assert (big[:, :, :, 50:] == 3.0).all()
    odd = torch.zeros((2, 3, 2, 50, 131), dtype=torch.bfloat16, device=DEV)
    kvquant.kvq_read(case.pool, case.dtable, case.dlens, 50, out=(odd[0, ..., 1:129], odd[1, ..., 1:129]))
    assert torch.equal(odd[0, ..., 1:129], k) and torch.equal(odd[1, ..., 1:129], v)
    assert torch.count_nonzero(odd[..., 0]) == 0 and torch.count_nonzero(odd[..., 129:]) == 0
    for b, n in enumerate(case.lens):
        assert torch.equal(k[b, :, :n].cpu(), case.k64[b].float().to(torch.bfloat16))
        assert torch.count_nonzero(k[b, :, n:]) == 0


# ------------------------------------------------------------------ the two in one launch
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 64)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("B,n,hq,hkv", [(3, 1, 8, 2), (2, 37, 5, 5), (40, 60, 16, 8)])
def test_append_qkv_equals_the_two_calls(fmt, D, rot, interleaved, B, n, hq, hkv):
    _need_gpu()
    from lara_b200 import kvquant, ops

    g = torch.Generator().manual_seed(B + n + D)
    ps, cap = 16, 160
    x = _rand_bf16(g, (B, n, hq + 2 * hkv, D))
    x[0, 0, hq, 5] = math.inf  # a k row that reads back as NaN
    x = x.to(DEV)
    q, k, v = x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:]
    starts = torch.randint(0, 90, (B,), generator=g).to(torch.int32)
    counts = torch.randint(0, n + 1, (B,), generator=g).to(torch.int32)
    counts[0] = n
    table, pages = _table(g, [cap] * B, cap // ps, ps)
    table, dstarts, dcounts = table.to(DEV), starts.to(DEV), counts.to(DEV)
    w = _rand_bf16(g, (2, D), False).to(DEV)
    tab = ops.rope_table(256, rot, device=DEV)
    pos = dstarts[:, None] + torch.arange(n, dtype=torch.int32, device=DEV)
    for norm, rope, odd in ((True, True, False), (True, False, False), (False, True, True), (False, False, False)):
        kw = dict(q_weight=w[0] if norm else None, k_weight=w[1] if norm else None, cos_sin=tab if rope else None,
                  interleaved=interleaved)
        pools = [kvquant.QuantPool.empty(pages, ps, hkv, D, fmt, DEV) for _ in range(2)]
        new = [torch.zeros(B, dtype=torch.int32, device=DEV) for _ in range(2)]
        qq, kk, vv = q, k, v
        if odd:
            qq, kk, vv = (torch.nn.functional.pad(z, (1, 2))[..., 1:D + 1] for z in (q, k, v))
        q2, k2 = ops.qk_norm_rope(q, k, positions=pos if rope else None, **kw) if norm or rope else (q, k)
        kvquant.kvq_append(pools[0], table, dstarts, k2.transpose(1, 2), v.transpose(1, 2), counts=dcounts,
                           new_lens=new[0])
        st = ops.new_workspace(256, DEV)
        q1 = kvquant.kvq_append_qkv(pools[1], table, dstarts, qq, kk, vv, counts=dcounts, new_lens=new[1],
                                    positions=pos if norm else None, workspace=st, **kw)
        assert ops.workspace_status(st) == 0
        assert torch.equal(q1, q2) and torch.equal(new[0], new[1])
        for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
            a, b = (getattr(p, name) for p in pools)
            if a.dtype == torch.float32:
                a, b = a.view(torch.int32), b.view(torch.int32)
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name


@pytest.mark.gpu
def test_append_qkv_reports_what_it_drops():
    _need_gpu()
    from lara_b200 import kvquant, ops

    pool = kvquant.QuantPool.empty(4, 16, 1, 64, "int8", DEV)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    table = i32([[0, 1], [2, 77]])
    g = torch.Generator().manual_seed(2)
    x = _rand_bf16(g, (2, 4, 3, 64)).to(DEV)
    st, new = ops.new_workspace(256, DEV), i32([0, 0])
    args = (x[:, :, :1], x[:, :, 1:2], x[:, :, 2:])
    tab = ops.rope_table(30, 64, device=DEV)
    kvquant.kvq_append_qkv(pool, table, i32([30, 14]), *args, cos_sin=tab, new_lens=new, workspace=st)
    assert ops.workspace_status(st) == 0x4 | 0x8 | 0x10  # past the capacity, page 77, positions past the table
    assert new.tolist() == [32, 18]
    kvquant.kvq_append_qkv(pool, table, i32([3, 4]), *(z[:, :0] for z in args), cos_sin=tab, new_lens=new,
                           workspace=st)
    assert ops.workspace_status(st) == 0 and new.tolist() == [3, 4]
    with pytest.raises(ValueError, match="shape"):
        kvquant.kvq_append_qkv(pool, table, i32([3, 4]), args[0], args[1], args[0][:, :1])


# ------------------------------------------------------------------ decode
LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 300, 777]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 8, 9, 16])
def test_decode_lengths(fmt, D, G):
    hkv = 2
    case = Case(LENS, hkv, D, 16 if G % 2 else 64, fmt, seed=G + D)
    g = torch.Generator().manual_seed(9)
    q = _rand_bf16(g, (len(LENS), hkv * G, D), False).to(DEV)
    o = _decode_gpu(case, q)
    case.check(q, o)
    assert torch.equal(o, _decode_gpu(case, q))  # the same words every time


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("B,hkv,n", [(1, 1, 5000), (1, 8, 3001), (3, 8, 1500), (70, 2, 200), (300, 1, 40)])
def test_decode_split_and_join(fmt, B, hkv, n):
    """Few long sequences (one head's tokens over many SMs) and many short ones."""
    g = torch.Generator().manual_seed(B + n)
    lens = torch.randint(1, n + 1, (B,), generator=g).tolist()
    lens[0] = n
    if B > 2:
        lens[B // 2] = 0
    case = Case(lens, hkv, 128, 64, fmt, seed=n)
    q = _rand_bf16(g, (B, hkv * 4, 128), False).to(DEV)
    o = _decode_gpu(case, q)
    case.check(q, o)
    assert torch.equal(o, _decode_gpu(case, q))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kind", ["peaked", "tiny_q", "huge_q", "late_max", "v_range", "zero_v", "explicit_scale"])
def test_decode_values(fmt, kind):
    g = torch.Generator().manual_seed(4)
    hkv, D, n = 2, 128, 400
    k, v = _rand_bf16(g, (1, hkv, n, D)), _rand_bf16(g, (1, hkv, n, D))
    q = _rand_bf16(g, (1, hkv * 4, D), False)
    scale = None
    if kind == "peaked":
        q = q * 8
    elif kind == "tiny_q":
        q = q * 2.0 ** -120
    elif kind == "huge_q":
        q = q * 2.0 ** 90
        k = k * 2.0 ** -90
    elif kind == "late_max":  # the largest scores come last, and grow
        k = (torch.arange(n).view(1, 1, n, 1) / n * 0.5 * q.view(1, hkv, 4, D)[:, :, :1]).to(torch.bfloat16)
    elif kind == "v_range":  # rows of V over 30 binary orders, the largest at unlikely tokens
        v = v * torch.exp2(torch.randint(-15, 15, (1, hkv, n, 1), generator=g).float())
    elif kind == "zero_v":
        v = torch.where(torch.rand((1, hkv, n, 1), generator=g) < 0.7, torch.zeros_like(v), v)
        v[:, 1] = 0
    else:
        scale = 0.31
    case = Case([n], hkv, D, 32, fmt, k_rows=k.to(torch.bfloat16), v_rows=v.to(torch.bfloat16))
    q = q.to(torch.bfloat16).to(DEV)
    case.check(q, _decode_gpu(case, q, scale=scale), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_nan_stays_where_it_is(fmt):
    """A NaN in q spoils its head alone, one in a cached row its kv head alone, one past the length nothing."""
    g = torch.Generator().manual_seed(8)
    hkv, D, n = 2, 64, 100
    k, v = _rand_bf16(g, (3, hkv, n, D)), _rand_bf16(g, (3, hkv, n, D))
    q = _rand_bf16(g, (3, hkv * 2, D), False)
    clean = Case([n] * 3, hkv, D, 16, fmt, k_rows=k, v_rows=v)
    o0 = _decode_gpu(clean, q.to(DEV))
    clean.check(q.to(DEV), o0)
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    q2[0, 1, 3] = math.nan
    k2[1, 0, 50, 9] = math.inf
    v2[2, 1, 99, 0] = math.nan
    o = _decode_gpu(Case([n] * 3, hkv, D, 16, fmt, k_rows=k2, v_rows=v2), q2.to(DEV))
    nan = torch.isnan(o)
    want = torch.zeros_like(nan)
    want[0, 1] = want[1, 0:2] = want[2, 2:4] = True
    assert torch.equal(nan, want)
    assert torch.equal(o[~want], o0[~want])


@pytest.mark.gpu
def test_decode_bad_page_and_length_are_reported():
    from lara_b200 import kvquant, ops

    case = Case([100, 40], 2, 128, 16, "int8", seed=2)
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=DEV)
    ws = kvquant.decode_workspace(2, 8, 2, 128, DEV)
    t = case.dtable.clone()
    t[0, 3] = 1000
    kvquant.gqa_decode_kvq(q, case.pool, t, case.dlens, workspace=ws)
    assert ops.workspace_status(ws) == 0x8
    for bad in (-1, 10 ** 6):
        lens = torch.tensor([100, bad], dtype=torch.int32, device=DEV)
        t2 = case.dtable.clamp_min(0)
        kvquant.gqa_decode_kvq(q, case.pool, t2, lens, workspace=ws)
        assert ops.workspace_status(ws) == 0x2
    o = kvquant.gqa_decode_kvq(q + 1, case.pool, case.dtable, case.dlens, workspace=ws)  # usable after that
    assert ops.workspace_status(ws) == 0
    case.check(q + 1, o)


@pytest.mark.gpu
def test_decode_shared_pages_and_streams_and_graph():
    """Two sequences share pages; the calls run on another stream and in a graph whose lengths change."""
    from lara_b200 import kvquant, ops

    case = Case([200, 200], 2, 128, 16, "int8", seed=12)
    case.table[1, :6] = case.table[0, :6]
    for x in (case.k64, case.v64):
        x[1][:, :96] = x[0][:, :96]
    case.dtable = case.table.to(DEV)
    g = torch.Generator().manual_seed(3)
    q = _rand_bf16(g, (2, 8, 128), False).to(DEV)
    case.check(q, _decode_gpu(case, q))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ws = kvquant.decode_workspace(2, 8, 2, 128, DEV)
    torch.cuda.synchronize()
    out = torch.empty_like(q)
    lens = case.dlens.clone()
    with torch.cuda.stream(side):
        for _ in range(2):
            kvquant.gqa_decode_kvq(q, case.pool, case.dtable, lens, workspace=ws, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kvquant.gqa_decode_kvq(q, case.pool, case.dtable, lens, workspace=ws, out=out)
    torch.cuda.synchronize()
    full = (case.k64, case.v64)
    for new in ([200, 200], [1, 0], [33, 150]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        case.lens = new
        case.k64, case.v64 = ([x[b][:, :n] for b, n in enumerate(new)] for x in full)
        case.check(q, out)
    assert ops.workspace_status(ws) == 0


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 codes: its last pages are written, read and attended."""
    _need_gpu()
    from lara_b200 import kvquant

    hkv, D, ps, n = 8, 128, 256, 300
    pages = (1 << 32) // (hkv * ps * D) + 8
    pool = kvquant.QuantPool.empty(pages, ps, hkv, D, "int8", DEV)
    table = torch.tensor([[pages - 1, 3], [0, pages - 2]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(0)
    k, v = _rand_bf16(g, (2, hkv, n, D)), _rand_bf16(g, (2, hkv, n, D))
    zero, lens = (torch.zeros(2, dtype=torch.int32, device=DEV) for _ in range(2))
    kvquant.kvq_append(pool, table, zero, k.to(DEV), v.to(DEV), new_lens=lens)
    ck, sk = quantise64(k, "int8")
    cv, sv = quantise64(v, "int8")
    kb, _ = kvquant.kvq_read(pool, table, lens, n)
    assert torch.equal(kb.cpu(), (ck.float() * sk.float()[..., None]).to(torch.bfloat16))
    q = _rand_bf16(g, (2, 32, D), False)
    o = kvquant.gqa_decode_kvq(q.to(DEV), pool, table, lens).double().cpu()
    k64, v64 = values64(ck, sk.float().double()), values64(cv, sv.float().double())
    for b in range(2):
        for h in range(hkv):
            ref, tol = attend64(q[b, 4 * h:4 * h + 4].double(), k64[b, h], v64[b, h], 1 / math.sqrt(D))
            assert ((o[b, 4 * h:4 * h + 4] - ref).abs() <= tol).all()


# ------------------------------------------------------------------ the cache manager
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_quant_cache_manager(tmp_path, fmt):
    _need_gpu()
    from lara_b200 import ops
    from lara_b200.kvquant import QuantKVCache

    g = torch.Generator().manual_seed(21)
    hkv, D, ps = 2, 128, 16
    c = QuantKVCache(num_pages=40, page_size=ps, n_kv_heads=hkv, head_dim=D, max_seqs=4, max_seq_len=256, fmt=fmt,
                     device=DEV)
    a, b = c.new_sequence(), c.new_sequence()
    k, v = _rand_bf16(g, (2, hkv, 70, D)), _rand_bf16(g, (2, hkv, 70, D))
    at = 0
    for n in (37, 1, 32):
        c.append(k[:, :, at:at + n].to(DEV), v[:, :, at:at + n].to(DEV), slots=[a, b])
        at += n
    s = c.new_sequence()
    assert c.share_prefix(a, s, 50) == 48
    c.append(k[1:, :, :5].to(DEV), v[1:, :, :5].to(DEV), slots=[s])
    assert [c.seq_len(x) for x in (a, b, s)] == [70, 70, 53]
    (ck, sk), (cv, sv) = quantise64(k, fmt), quantise64(v, fmt)
    k64, v64 = values64(ck, sk.float().double()), values64(cv, sv.float().double())
    ks = [k64[0], k64[1], torch.cat([k64[0, :, :48], k64[1, :, :5]], 1)]
    vs = [v64[0], v64[1], torch.cat([v64[0, :, :48], v64[1, :, :5]], 1)]
    kb, vb = c.read()
    for i in range(3):
        n = ks[i].shape[1]
        assert torch.equal(kb[i, :, :n].cpu(), ks[i].float().to(torch.bfloat16))
        assert torch.count_nonzero(kb[i, :, n:]) == 0
        assert torch.equal(c.gather([a, b, s][i])[1], vb[i, :, :n])
    q = _rand_bf16(g, (3, hkv * 4, D), False)
    o = c.decode(q.to(DEV)).double().cpu()
    for i in range(3):
        for h in range(hkv):
            ref, tol = attend64(q[i, 4 * h:4 * h + 4].double(), ks[i][h], vs[i][h], 1 / math.sqrt(D))
            assert ((o[i, 4 * h:4 * h + 4] - ref).abs() <= tol).all()
    assert c.status() == 0
    # a file holds the values; quantising them again gives the same ones
    c.save(tmp_path / "c.npz")
    d = QuantKVCache(num_pages=40, page_size=32, n_kv_heads=hkv, head_dim=D, max_seqs=4, max_seq_len=256, fmt=fmt,
                     device=DEV)
    assert d.load(tmp_path / "c.npz") == [0, 1, 2]
    assert torch.equal(d.read()[0], kb) and torch.equal(d.read()[1], vb)
    # chunked prefill over the quantised prefix: read it into a bf16 cache, append, attend
    kc, vc = (torch.zeros((3, hkv, 96, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    c.read(out=(kc[:, :, :70], vc[:, :, :70]))
    new = _rand_bf16(g, (3, hkv, 8, D)).to(DEV)
    lens = torch.tensor([70, 70, 53], dtype=torch.int32, device=DEV)
    cached = lens.clone()
    ops.kv_append(kc, vc, lens, new, new)
    out = ops.gqa_prefill(_rand_bf16(g, (3, 8, hkv * 4, D)).to(DEV), kc, vc, cached)
    assert torch.isfinite(out).all()
    for x in (a, b, s):
        c.free_sequence(x)
    assert c.free_pages == c.num_pages


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotation_alone_keeps_infinities_apart(interleaved):
    """Without a norm, dims past rot_dim pass through, infinities and NaN beside them or not."""
    _need_gpu()
    from lara_b200 import ops

    g = torch.Generator().manual_seed(13)
    x = _rand_bf16(g, (9, 3, 128))
    x[1, 0, 70], x[2, 1, 127], x[3, 2, 96] = math.inf, -math.inf, math.nan
    pos = torch.arange(9, dtype=torch.int32, device=DEV)
    q, k = ops.qk_norm_rope(x.to(DEV), x[:, :1].to(DEV), positions=pos, cos_sin=ops.rope_table(9, 64, device=DEV),
                            interleaved=interleaved)
    for y in (q, k):
        h = y.shape[1]
        got, want = y[..., 64:].cpu(), x[:, :h, 64:]
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(7.0, math.inf, -math.inf), want.nan_to_num(7.0, math.inf, -math.inf))
        assert torch.isfinite(y[..., :64]).all()


@pytest.mark.gpu
def test_small_batches_and_empty_calls():
    _need_gpu()
    from lara_b200 import kvquant, ops

    case = Case([5, 3], 2, 64, 16, "fp8_e4m3", seed=1)
    q = torch.empty((0, 4, 64), dtype=torch.bfloat16, device=DEV)
    none = torch.empty((0,), dtype=torch.int32, device=DEV)
    assert kvquant.gqa_decode_kvq(q, case.pool, case.dtable[:0], none).shape == (0, 4, 64)
    k, v = kvquant.kvq_read(case.pool, case.dtable[:0], none, 7)
    assert k.shape == v.shape == (0, 2, 7, 64)
    kvquant.kvq_append(case.pool, case.dtable[:0], none, k, v)
    a, b = ops.qk_norm_rope(q, q[:, :1], q_weight=torch.ones(64, dtype=torch.bfloat16, device=DEV),
                            k_weight=torch.ones(64, dtype=torch.bfloat16, device=DEV))
    assert a.shape == (0, 4, 64) and b.shape == (0, 1, 64)
    with pytest.raises(ValueError, match="seq_lens"):
        kvquant.kvq_read(case.pool, case.dtable, case.dlens.long(), 7)
    with pytest.raises(ValueError, match="block_table"):
        kvquant.kvq_read(case.pool, case.dtable[:1], case.dlens, 7)
    with pytest.raises(ValueError, match="stride of 0"):
        z = torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16, device=DEV).expand(2, 2, 7, 64)
        kvquant.kvq_read(case.pool, case.dtable, case.dlens, 7, out=(z, z))
    with pytest.raises(ValueError, match="shape"):
        kvquant.gqa_decode_kvq(torch.zeros((2, 4, 128), dtype=torch.bfloat16, device=DEV), case.pool, case.dtable,
                               case.dlens)


@pytest.mark.gpu
def test_small_workspaces_and_odd_flags_are_refused():
    _need_gpu()
    from lara_b200 import kvquant, ops

    case = Case([5, 3], 2, 64, 16, "int8", seed=1)
    small = torch.zeros(255, dtype=torch.uint8, device=DEV)
    k = torch.zeros((2, 2, 1, 64), dtype=torch.bfloat16, device=DEV)
    heads = torch.zeros((2, 1, 2, 64), dtype=torch.bfloat16, device=DEV)
    for call in (lambda ws: kvquant.kvq_read(case.pool, case.dtable, case.dlens, 7, workspace=ws),
                 lambda ws: kvquant.kvq_append(case.pool, case.dtable, case.dlens, k, k, workspace=ws),
                 lambda ws: kvquant.kvq_append_qkv(case.pool, case.dtable, case.dlens, heads, heads, heads, workspace=ws),
                 lambda ws: ops.qk_norm_rope(heads, heads, workspace=ws)):
        for ws in (small, small[:0], torch.zeros(400, dtype=torch.uint8, device=DEV)[1:300]):
            with pytest.raises(ValueError, match="256 bytes"):
                call(ws)
    for call in (lambda flag: ops.qk_norm_rope(heads, heads, interleaved=flag),
                 lambda flag: kvquant.kvq_append_qkv(case.pool, case.dtable, case.dlens, heads, heads, heads,
                                                     interleaved=flag)):
        with pytest.raises(TypeError, match="truth value"):
            call(torch.zeros(2))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,G", [(128, 4), (128, 12), (64, 8), (64, 16)])
@pytest.mark.parametrize("B,hkv,n", [(150, 8, 100), (80, 8, 700), (7, 4, 3000), (1300, 1, 60), (1300, 1, 900)])
def test_decode_shares(fmt, D, G, B, hkv, n):
    """More (sequence, kv head) units than CTAs, short and long, and few long ones; ragged, some empty."""
    g = torch.Generator().manual_seed(B + D + G)
    lens = torch.randint(1, n + 1, (B,), generator=g).tolist()
    lens[0], lens[3], lens[B - 1] = n, 0, 1
    lens[4:6] = [0, 0]
    # the same rows for every sequence keep the reference quick; their pages are their own
    k, v = _rand_bf16(g, (1, hkv, n, D)), _rand_bf16(g, (1, hkv, n, D))
    case = SharedRows(lens, hkv, D, 64, fmt, k[0], v[0], seed=n)
    q = _rand_bf16(g, (B, hkv * G, D), False).to(DEV)
    o = _decode_gpu(case, q)
    case.check(q, o)
    assert torch.equal(o, _decode_gpu(case, q))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,G", [(128, 5), (128, 16), (64, 8), (64, 9)])
@pytest.mark.parametrize("B,hkv,n,filled", [(90, 8, 510, 90), (41, 16, 512, 40), (900, 1, 700, 66), (700, 1, 480, 699)])
def test_decode_whole_units(fmt, D, G, B, hkv, n, filled):
    """Units too short to be cut, more than CTAs; and fewer, of a batch that is mostly empty."""
    g = torch.Generator().manual_seed(B + D + G)
    lens = torch.zeros(B, dtype=torch.int64)
    lens[torch.randperm(B, generator=g)[:filled]] = torch.randint(n // 2, n + 1, (filled,), generator=g)
    lens = lens.tolist()
    k, v = _rand_bf16(g, (1, hkv, n, D)), _rand_bf16(g, (1, hkv, n, D))
    case = SharedRows(lens, hkv, D, 32, fmt, k[0], v[0], seed=n)
    q = _rand_bf16(g, (B, hkv * G, D), False).to(DEV)
    o = _decode_gpu(case, q)
    case.check(q, o)
    assert torch.equal(o, _decode_gpu(case, q))


class SharedRows(Case):
    """Every sequence holds the first rows of one K and V; written page by page."""

    def __init__(self, lens, hkv, D, ps, fmt, k, v, seed=0):
        from lara_b200 import kvquant

        _need_gpu()
        g = torch.Generator().manual_seed(seed)
        self.lens, self.fmt, self.D, self.hkv, self.ps = list(lens), fmt, D, hkv, ps
        n = max(lens)
        per_seq = -(-n // ps)
        self.table, pages = _table(g, lens, per_seq, ps)
        pools, self.k64, self.v64 = [], [], []
        for x, keep in ((k, self.k64), (v, self.v64)):
            c, s = quantise64(torch.nn.functional.pad(x, (0, 0, 0, per_seq * ps - n)), fmt)
            keep += [values64(c, s.float().double())[:, :m] for m in lens]
            bits = (c.to(torch.int8) if fmt == "int8" else c.float().to(torch.float8_e4m3fn)).view(torch.uint8)
            codes = torch.zeros((pages, hkv, ps, D), dtype=torch.uint8)
            scales = torch.zeros((pages, hkv, ps))
            for b, m in enumerate(lens):
                for j in range(-(-m // ps)):
                    p = int(self.table[b, j])
                    codes[p] = bits[:, j * ps:(j + 1) * ps]
                    scales[p] = s[:, j * ps:(j + 1) * ps].float()
            pools.append((codes.to(DEV).view(DTYPES[fmt]), scales.to(DEV)))
        self.pool = kvquant.QuantPool(pools[0][0], pools[1][0], pools[0][1], pools[1][1])
        self.dtable = self.table.to(DEV)
        self.dlens = torch.tensor(self.lens, dtype=torch.int32, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,bound", [("int8", 0.02), ("fp8_e4m3", 0.08)])
def test_example_runs_them_together(fmt, bound):
    """``examples/quantised_cache.py``: prompts, then steps from a CUDA graph.

    The bounds are the formats' own errors: int8 rounds to 1/254 of a row's largest value (about 3 of a normal
    row's deviations), 0.7 % of a value's deviation in K and V; e4m3 to 2^-4, 2.6 % on average; each counts in the
    weights and in the values, with a factor of two for the worst sequence and a little for bf16.
    """
    _need_gpu()
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location(
        "quantised_cache", Path(__file__).resolve().parents[1] / "examples" / "quantised_cache.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    r = mod.run(fmt=fmt, batch=5, prompt=200, steps=7)
    assert r["status"] == 0
    assert r["lens"] == r["expected_lens"]
    assert r["relative_error"] < bound


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 5, 900])
def test_decode_of_empty_sequences_alone(B):
    case = SharedRows([1] * B, 1, 128, 16, "int8", torch.zeros((1, 1, 128)), torch.zeros((1, 1, 128)))
    from lara_b200 import kvquant, ops

    ws = kvquant.decode_workspace(B, 4, 1, 128, DEV)
    q = torch.ones((B, 4, 128), dtype=torch.bfloat16, device=DEV)
    out = torch.full_like(q, 3.0)
    kvquant.gqa_decode_kvq(q, case.pool, case.dtable, torch.zeros_like(case.dlens), workspace=ws, out=out)
    assert ops.workspace_status(ws) == 0 and torch.count_nonzero(out) == 0


@pytest.mark.gpu
def test_int8_codes_of_every_ratio():
    """Every pair of bf16 significands and 20 exponents apart: the code is the exact quotient's, ties to even."""
    _need_gpu()
    from lara_b200 import kvquant

    top = torch.arange(128, 256, dtype=torch.float64)                      # a
    x = (torch.arange(128, 256, dtype=torch.float64)[None, :] * 2.0 ** -torch.arange(0, 20, dtype=torch.float64)[:, None])
    x = torch.cat([x.flatten(), -x.flatten()])                             # 5120 values
    per = 127
    n = -(-x.numel() // per)
    xs = torch.nn.functional.pad(x, (0, n * per - x.numel())).view(n, per)
    for scale in (2.0 ** -100, 2.0 ** -40, 1.0, 2.0 ** 115):
        k = torch.zeros((128, 1, n, 128), dtype=torch.float64)
        k[..., 0] = top[:, None, None]
        k[..., 1:] = torch.where(xs.abs()[None] <= top[:, None, None], xs[None], 0.0)[:, None]
        k = (k * scale).to(torch.bfloat16)
        pages = 128 * (-(-n // 16))
        pool = kvquant.QuantPool.empty(pages, 16, 1, 128, "int8", DEV)
        table = torch.arange(pages, dtype=torch.int32, device=DEV).view(128, -1)
        zero = torch.zeros(128, dtype=torch.int32, device=DEV)
        kvquant.kvq_append(pool, table, zero, k.to(DEV), k.to(DEV))
        c64, s64 = quantise64(k, "int8")
        codes = pool.k_codes.view(128, -1, 128)[:, :n].cpu()
        assert torch.equal(codes, c64[:, 0].to(torch.int8))
        assert torch.equal(pool.k_scales.view(128, -1)[:, :n].cpu(), s64[:, 0].float())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,hkv,G,D", [([140000], 1, 2, 64), ([40000, 3, 0], 1, 4, 128), ([9000] * 4, 1, 16, 128)])
def test_decode_few_long_sequences(fmt, lens, hkv, G, D):
    """Units that many CTAs share: joined in one step, and in two."""
    g = torch.Generator().manual_seed(len(lens) + G)
    n = max(lens)
    k, v = _rand_bf16(g, (hkv, n, D)), _rand_bf16(g, (hkv, n, D))
    case = SharedRows(lens, hkv, D, 256, fmt, k, v, seed=n)
    q = _rand_bf16(g, (len(lens), hkv * G, D), False).to(DEV)
    o = _decode_gpu(case, q)
    case.check(q, o)
    assert torch.equal(o, _decode_gpu(case, q))
