"""Every way in which the 8-bit KV cache operators and the q/k head pass share out, hold or access their work.

Decode outputs are checked element by element (``attend64_close``) and by the norm of each head's error: 2^-8 of the
head's norm, which the bf16 rounding of the output alone stays under on any head (at 0.45 of it on ordinary ones).
Unlike bounds that grow with the number of tokens it fails for a lost tile of 32 of them among 140000: of unit normal
rows, such as all of these tests have, its share of a head's norm is sqrt(32 / 140000) = 2^-6.
"""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_kvquant import (DEV, FORMATS, SharedRows, _decode_gpu, _rand_bf16, _table, norm_rope64,  # noqa: E402
                          quantise64, values64)
from test_kvquant_bounds import check_close  # noqa: E402


def _rows(g, *shape):
    return _rand_bf16(g, shape, outliers=False)


def norm_error(got, ref):
    """The largest relative error, in norm, of the heads got, ref [G, D]."""
    got, ref = got.double().cpu(), ref.double().cpu()
    return float(((got - ref).norm(dim=-1) / ref.norm(dim=-1)).max())


BOUND = 2.0 ** -8


def check_norms(case, q, o):
    q, o = q.double().cpu(), o.double().cpu()
    G = q.shape[1] // case.hkv
    for b, n in enumerate(case.lens):
        for h in range(case.hkv):
            if n:
                s = slice(h * G, (h + 1) * G)
                ref = torch.softmax((q[b, s] @ case.k64[b][h].T) / case.D ** 0.5, -1) @ case.v64[b][h]
                assert norm_error(o[b, s], ref) <= BOUND, (b, h, n)


@pytest.mark.parametrize("fmt", FORMATS)
def test_the_norm_bound_sees_lost_tokens(fmt):
    """At the length and heads of the longest join: zeros, half of the tokens, a CTA's part, a warp's tile, a warp."""
    g = torch.Generator().manual_seed(1)
    n, G, D = 140000, 2, 64
    k, v = (values64(*[x.double() for x in quantise64(_rows(g, n, D), fmt)]) for _ in range(2))
    q = _rows(g, G, D).double()
    p = torch.exp(q @ k.T / D ** 0.5)

    def out(keep):
        w = p * keep
        return (w @ v) / w.sum(-1, keepdim=True)

    all_ = torch.ones(n, dtype=torch.float64)
    ref = out(all_)
    assert norm_error(ref.to(torch.bfloat16), ref) <= 0.6 * BOUND
    assert norm_error(torch.zeros_like(ref), ref) > BOUND
    for lo, hi in ((0, n // 2), (64000, 64000 + 256), (139968, n), (0, 32), (70016, 70048)):
        keep = all_.clone()
        keep[lo:hi] = 0
        assert norm_error(out(keep).to(torch.bfloat16), ref) > BOUND, (lo, hi)
    tiles = (torch.arange(n) // 32) % 4
    assert norm_error(out((tiles != 2).double()).to(torch.bfloat16), ref) > BOUND


# ------------------------------------------------------------------ decode: parts of a unit
def parts_of_longest(lens, hkv, G, D):
    """CTAs that share the longest sequence's first kv head where shares are cut across units; None elsewhere.

    The rules of kvq_decode.cu restated: tiles of 32 tokens, an extra cost per unit, equal shares.
    """
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    ng = 1 if G <= 8 else 2
    grid = sms * {(128, 1): 3, (128, 2): 2, (64, 1): 4, (64, 2): 3}[D, ng]
    tiles = [-(-n // 32) for n in lens]
    longest, total = max(tiles), sum(tiles) * hkv
    units = sum(t > 0 for t in tiles) * hkv
    if longest <= 24 or units * 8 <= grid:
        return None
    gap = 8 * ng
    span = total + units * gap
    workers = min(grid, max(-(-total // 4), units))
    per, rem = divmod(span, workers)

    def cta(x):
        return x // (per + 1) if x < rem * (per + 1) else rem + (x - rem * (per + 1)) // per

    b = tiles.index(longest)
    first = (sum(tiles[:b]) + sum(t > 0 for t in tiles[:b]) * gap) * hkv + gap
    return cta(first + longest - 1) - cta(first) + 1


def _mixed(B, n, long, at):
    g = torch.Generator().manual_seed(B + long)
    lens = torch.randint(n // 2, n + 1, (B,), generator=g).tolist()
    lens[at], lens[0 if at else 1] = long, 0
    return lens


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("G,D", [(4, 128), (16, 128), (4, 64), (16, 64)])
@pytest.mark.parametrize("B,n,long,at,few", [(90, 300, 100000, 7, 65), (90, 300, 100000, 89, 65), (90, 300, 8000, 40, 5),
                                             (200, 2000, 30000, 0, 5), (400, 1500, 1500, 3, 1)])
def test_decode_shares_cut_across_units(fmt, G, D, B, n, long, at, few):
    """One sequence among many shorter ones over 1 to 4, 5 to 64, and more CTAs; the last are joined in two steps."""
    lens = _mixed(B, n, long, at)
    parts = parts_of_longest(lens, 1, G, D)
    assert few <= parts and (few != 5 or parts <= 64) and (few != 1 or parts <= 4), parts
    g = torch.Generator().manual_seed(G + D)
    case = SharedRows(lens, 1, D, 64, fmt, _rows(g, 1, max(lens), D), _rows(g, 1, max(lens), D), seed=B)
    q = _rows(g, B, G, D).to(DEV)
    o = _decode_gpu(case, q)
    check_norms(case, q, o)
    check_close(case, q, o, chain=4 * 64 + 128)  # at most 64 tiles of a warp, 4 products each; the joins
    assert torch.equal(o, _decode_gpu(case, q))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,hkv,G,D", [([140000], 1, 2, 64), ([140000], 1, 2, 128), ([300000], 1, 16, 128),
                                          ([40000, 3, 0], 1, 4, 128), ([9000] * 4, 1, 16, 128), ([3001], 8, 4, 128),
                                          ([5000], 1, 4, 128), ([1500, 700, 1], 8, 4, 64), ([262144], 2, 16, 128)])
def test_decode_few_units(fmt, lens, hkv, G, D):
    """Units with CTAs of their own, joined in one step and in two."""
    g = torch.Generator().manual_seed(len(lens) + G)
    n = max(lens)
    case = SharedRows(lens, hkv, D, 256, fmt, _rows(g, hkv, n, D), _rows(g, hkv, n, D), seed=n)
    q = _rows(g, len(lens), hkv * G, D).to(DEV)
    o = _decode_gpu(case, q)
    check_norms(case, q, o)
    check_close(case, q, o, chain=4 * 64 + 128)
    assert torch.equal(o, _decode_gpu(case, q))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("G,D", [(5, 128), (12, 128), (8, 64), (9, 64)])
@pytest.mark.parametrize("B,hkv,n", [(16, 2, 777), (150, 8, 100), (80, 8, 700), (1300, 1, 60), (2400, 1, 500)])
def test_decode_norms_of_other_shares(fmt, G, D, B, hkv, n):
    """A CTA for each unit, units to warps, to CTAs whole."""
    g = torch.Generator().manual_seed(B + D + G)
    lens = torch.randint(1, n + 1, (B,), generator=g).tolist()
    case = SharedRows(lens, hkv, D, 64, fmt, _rows(g, hkv, n, D), _rows(g, hkv, n, D), seed=n)
    q = _rows(g, B, hkv * G, D).to(DEV)
    o = _decode_gpu(case, q)
    check_norms(case, q, o)
    check_close(case, q, o, chain=4 * 24 + 128)


# ------------------------------------------------------------------ q/k head pass: heads per lane group
def _fill(tokens, heads, D):
    return tokens * heads * (D // 8) / (torch.cuda.get_device_properties(0).multi_processor_count * 2048.0)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 72), (64, 32)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("fill", [0.3, 1.0, 2.5, 5.0])
@pytest.mark.parametrize("hq,hkv", [(13, 3), (8, 8)])
def test_norm_rope_heads_per_lane_group(D, rot, interleaved, fill, hq, hkv):
    """One, two, four and eight heads, the last group of q and k not full; in 64 bits, on the tests' own bound."""
    from lara_b200 import ops

    T = int(fill * 148 * 2048 / ((hq + hkv) * (D // 8))) + 1
    assert 0.9 * fill <= _fill(T, hq + hkv, D) <= 1.1 * fill
    g = torch.Generator().manual_seed(T + D)
    q, k = (_rand_bf16(g, (T, h, D)).to(DEV) for h in (hq, hkv))
    qw, kw = (_rows(g, D).to(DEV) for _ in range(2))
    pos = torch.randint(0, 5000, (T,), generator=g).to(torch.int32).to(DEV)
    tab = ops.rope_table(5000, rot, device=DEV)
    cs = tab[pos.long()]
    for norm in (True, False):
        got = ops.qk_norm_rope(q, k, positions=pos, cos_sin=tab, q_weight=qw if norm else None,
                               k_weight=kw if norm else None, interleaved=interleaved)
        for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
            ref, mag = norm_rope64(x, w if norm else None, cs[:, :rot // 2], cs[:, rot // 2:], interleaved, 1e-5)
            err = (y.double() - ref).abs()
            assert int((err > 2.0 ** -8 * ref.abs() + 16 * 2.0 ** -24 * mag + 2.0 ** -133).sum()) == 0


# ------------------------------------------------------------------ rows that start on 16-byte boundaries
def _half_aligned(x):
    """x, its rows on 16-byte boundaries that are not 32-byte ones."""
    y = torch.zeros((*x.shape[:-1], x.shape[-1] + 16), dtype=x.dtype, device=DEV)[..., 8:x.shape[-1] + 8]
    y.copy_(x)
    assert y.data_ptr() % 32 == 16 and all(s * 2 % 32 == 0 for s in y.stride()[:-1])
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
def test_append_and_read_of_half_aligned_rows(fmt, D):
    from lara_b200 import kvquant

    g = torch.Generator().manual_seed(D)
    B, hkv, n, ps = 3, 3, 41, 16
    x = [_rand_bf16(g, (B, hkv, n, D)) for _ in range(2)]
    lens = [n] * B
    table, pages = _table(g, lens, -(-n // ps), ps)
    pool = kvquant.QuantPool.empty(pages, ps, hkv, D, fmt, DEV)
    zero = torch.zeros(B, dtype=torch.int32, device=DEV)
    kvquant.kvq_append(pool, table.to(DEV), zero, *(_half_aligned(t) for t in x))
    full = torch.full_like(zero, n)
    out = tuple(_half_aligned(torch.zeros((B, hkv, n, D), dtype=torch.bfloat16)) for _ in range(2))
    kvquant.kvq_read(pool, table.to(DEV), full, n, out=out)
    for t, y in zip(x, out):
        c, s = quantise64(t, fmt)
        assert torch.equal(y.cpu(), (c.float() * s.float()[..., None]).to(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 72), (64, 64)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("B,n,hq,hkv", [(3, 5, 13, 3), (40, 130, 13, 3)])
@pytest.mark.parametrize("half", [False, True])
def test_append_qkv_in_64_bits(fmt, D, rot, interleaved, B, n, hq, hkv, half):
    """One and four heads per lane group, the last not full, rows on 32- and 16-byte boundaries.

    q against its definition; the stored k and v against those of a separate append of what the pass makes of k, and
    that against the definition.
    """
    from lara_b200 import kvquant, ops

    g = torch.Generator().manual_seed(B + n + D)
    ps, pps = 64, 4
    q, k, v = (_rand_bf16(g, (B, n, h, D)).to(DEV) for h in (hq, hkv, hkv))
    args = [_half_aligned(t) if half else t for t in (q, k, v)]
    w = [_rows(g, D).to(DEV) for _ in range(2)]
    tab = ops.rope_table(400, rot, device=DEV)
    starts = torch.randint(0, 100, (B,), generator=g).to(torch.int32).to(DEV)
    pos = starts[:, None] + torch.arange(n, dtype=torch.int32, device=DEV)
    cs = tab[pos.long()]
    table = torch.randperm(B * pps, generator=g).to(torch.int32).view(B, pps).to(DEV)
    pool, other = (kvquant.QuantPool.empty(B * pps, ps, hkv, D, fmt, DEV) for _ in range(2))
    new, st = torch.zeros_like(starts), ops.new_workspace(256, DEV)
    kw = dict(cos_sin=tab, q_weight=w[0], k_weight=w[1], interleaved=interleaved)
    out = _half_aligned(torch.zeros_like(q)) if half else None
    got = kvquant.kvq_append_qkv(pool, table, starts, *args, new_lens=new, workspace=st, out=out, **kw)
    assert ops.workspace_status(st) == 0
    _, turned = ops.qk_norm_rope(q, k, positions=pos, **kw)
    for x, wt, y in ((q, w[0], got), (k, w[1], turned)):
        ref, mag = norm_rope64(x, wt, cs[..., :rot // 2], cs[..., rot // 2:], interleaved, 1e-5)
        err = (y.double() - ref).abs()
        assert int((err > 2.0 ** -8 * ref.abs() + 16 * 2.0 ** -24 * mag + 2.0 ** -133).sum()) == 0
    kvquant.kvq_append(other, table, starts, turned.transpose(1, 2), v.transpose(1, 2))
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        assert torch.equal(getattr(pool, name).view(torch.uint8), getattr(other, name).view(torch.uint8)), name
    back = kvquant.kvq_read(pool, table, new, n, starts=starts)
    for x, y in zip((turned, v), back):
        c, s = quantise64(x.transpose(1, 2).cpu(), fmt)
        assert torch.equal(y.cpu(), (c.float() * s.float()[..., None]).to(torch.bfloat16))


# ------------------------------------------------------------------ the documented loop
@pytest.mark.gpu
def test_the_documented_serving_loop():
    """The integration guide's loop over views of one projection output: every step appends behind the last one's token."""
    import re
    from pathlib import Path

    from lara_b200 import kvquant, ops

    text = (Path(__file__).resolve().parents[1] / "INTEGRATION.md").read_text()
    code = next(c for c in re.findall(r"```python\n(.*?)```", text, re.S) if "decode_workspace" in c)
    B, Hq, Hkv, D, ps = 3, 8, 2, 64, 16
    g = torch.Generator().manual_seed(5)
    x = _rows(g, B, 1, Hq + 2 * Hkv, D).to(DEV)
    q, k, v = x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]
    pool = kvquant.QuantPool.empty(12, ps, Hkv, D, "int8", DEV)
    table = torch.arange(12, dtype=torch.int32, device=DEV).view(B, 4)
    lens = torch.tensor([0, 15, 20], dtype=torch.int32, device=DEV)
    want = [int(n) for n in lens]
    env = dict(torch=torch, kvquant=kvquant, ops=ops, B=B, Hq=Hq, Hkv=Hkv, D=D, pool=pool, block_table=table, lens=lens,
               q=q, k=k, v=v, o=torch.empty((B, Hq, D), dtype=torch.bfloat16, device=DEV),
               cos_sin=ops.rope_table(64, D, device=DEV))
    exec(code, env)
    for _ in range(2):
        env["step"]()
    assert lens.tolist() == [n + 3 for n in want]
    vb = kvquant.kvq_read(pool, table, lens, 23)[1]
    c, s = quantise64(v[:, 0].cpu(), "int8")
    row = (c.float() * s.float()[..., None]).to(torch.bfloat16).to(DEV)
    for b, n in enumerate(want):
        for t in range(n, n + 3):
            assert torch.equal(vb[b, :, t], row[b])
    assert torch.isfinite(env["o"]).all()
