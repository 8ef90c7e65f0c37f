"""Closer checks of the 8-bit KV cache operators and the q/k head pass than worst-case sums over all tokens.

``attend64_close`` bounds the decode by what its sums are: a weight is two fp16 numbers (2^-20 of itself, the
exponential's error with it), a score 136 fp32 roundings (2^-24 of ``sum_d |q_d k_d|``, twice: above and below the
line), the sums over tokens chains of ``chain`` fp32 additions (2^-23 of ``kappa = sum_t p_t |v_t|``), weights too
small for fp16's last place 2^-30 of the row's largest kappa each, and one bf16 rounding at the end (2^-8).
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from test_kvquant import DEV, FORMATS, Case, SharedRows, _decode_gpu, _rand_bf16  # noqa: E402


# ------------------------------------------------------------------ bounds
def attend64_close(q, k, v, scale, chain):
    """q [G, D], k/v [n, D] float64 -> (o [G, D], absolute tolerance [G, D])."""
    n = k.shape[0]
    s = (q @ k.T) * scale
    mag = (q.abs() @ k.abs().T) * scale
    p = torch.softmax(s, -1)
    o, kappa = p @ v, p @ v.abs()
    rel = 2.0 ** -20 + 2 * 136 * 2.0 ** -24 * mag.amax(-1, keepdim=True) + chain * 2.0 ** -23
    return o, 2.0 ** -8 * o.abs() + rel * kappa + n * 2.0 ** -30 * kappa.amax(-1, keepdim=True) + 2.0 ** -133


def check_close(case, q, o, chain, scale=None):
    sc = 1.0 / math.sqrt(case.D) if scale is None else scale
    G = q.shape[1] // case.hkv
    o, q = o.double().cpu(), q.double().cpu()
    for b, n in enumerate(case.lens):
        for h in range(case.hkv):
            got = o[b, h * G:(h + 1) * G]
            if n == 0:
                assert torch.count_nonzero(got) == 0
                continue
            ref, tol = attend64_close(q[b, h * G:(h + 1) * G], case.k64[b][h], case.v64[b][h], sc, chain)
            assert ((got - ref).abs() <= tol).all(), (b, h, n, ((got - ref).abs() / tol).max())


# ------------------------------------------------------------------ decode
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,G", [(128, 1), (128, 4), (128, 8), (128, 16), (64, 3), (64, 9)])
def test_decode_weights_keep_more_than_fp16(fmt, D, G):
    """Two tokens of nearly equal weight and opposite values: what is left is the weights' difference.

    Scores of a few tenths out of two dims, so that their roundings stay below those of an fp16 weight.
    """
    g = torch.Generator().manual_seed(D + G)
    B, hkv = 40, 2
    k = torch.zeros((B, hkv, 2, D))
    k[..., 0] = 1.0
    k[..., 1] = torch.randint(-2, 3, (B, hkv, 2), generator=g) * 2.0 ** -6
    v = _rand_bf16(g, (B, hkv, 1, D)).float()
    case = Case([2] * B, hkv, D, 16, fmt, k_rows=k.to(torch.bfloat16), v_rows=torch.cat([v, -v], 2).to(torch.bfloat16))
    q = (0.2 * torch.randn((B, hkv * G, D), generator=g) * math.sqrt(D)).to(torch.bfloat16).to(DEV)
    check_close(case, q, _decode_gpu(case, q), chain=8)


# ------------------------------------------------------------------ append: grids of more than 2^31 threads
def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _large_batch(B):
    """starts 0 .. 14, counts 0 but for a few, a table whose every sequence has page 0, and those with rows their own."""
    starts = torch.arange(B, dtype=torch.int32, device=DEV) % 15
    counts = torch.zeros(B, dtype=torch.int32, device=DEV)
    table = torch.zeros((B, 1), dtype=torch.int32, device=DEV)
    some = [0, 1, B // 2, B - 2, B - 1]
    counts[some] = 1
    table[some, 0] = torch.arange(len(some), dtype=torch.int32, device=DEV)
    return starts, counts, table, some


@pytest.mark.gpu
def test_append_lengths_of_a_large_grid():
    """One row each of 2^26 - 1 sequences: the grid has 2^31 threads, and each length is written once."""
    from lara_b200 import kvquant, ops

    B = 2 ** 26 - 1
    starts, counts, table, some = _large_batch(B)
    pool = kvquant.QuantPool.empty(len(some), 16, 1, 64, "int8", DEV)
    row = torch.arange(64, device=DEV).to(torch.bfloat16)
    x = row.expand(B, 1, 1, 64)
    new, st = torch.full_like(starts, -7), ops.new_workspace(256, DEV)
    kvquant.kvq_append(pool, table, starts, x, x, counts=counts, new_lens=new, workspace=st)
    assert ops.workspace_status(st) == 0
    assert torch.equal(new, starts + counts)
    for i, b in enumerate(some):
        at = int(starts[b])
        assert torch.count_nonzero(pool.k_scales[i, 0]) == 1 and torch.count_nonzero(pool.v_codes[i, 0].sum(-1)) == 1
        assert torch.equal(pool.k_codes[i, 0, at], torch.round(127.0 * row.float() / 63.0).to(torch.int8))


@pytest.mark.gpu
def test_append_qkv_lengths_of_a_large_grid():
    """One token each of 2^27 sequences, three heads of sixteen lanes: more than 2^32 threads."""
    from lara_b200 import kvquant, ops

    B, D = 2 ** 27, 128
    starts, counts, table, some = _large_batch(B)
    pool = kvquant.QuantPool.empty(len(some), 16, 1, D, "int8", DEV)
    row = torch.arange(D, device=DEV).to(torch.bfloat16)
    x = row.expand(B, 1, 1, D)
    out = torch.empty((B, 1, 1, D), dtype=torch.bfloat16, device=DEV)
    tab = torch.cat([torch.ones((16, 4), device=DEV), torch.zeros((16, 4), device=DEV)], -1)  # a turn by nothing
    new, st = torch.full_like(starts, -7), ops.new_workspace(256, DEV)
    kvquant.kvq_append_qkv(pool, table, starts, x, x, x, cos_sin=tab, counts=counts, new_lens=new, workspace=st, out=out)
    assert ops.workspace_status(st) == 0
    assert torch.equal(new, starts + counts)
    for i, b in enumerate(some):
        assert torch.equal(out[b, 0, 0], row)
        assert torch.count_nonzero(pool.k_scales[i, 0]) == 1
        assert torch.equal(pool.k_codes[i, 0, int(starts[b])], torch.round(127.0 * row.float() / 127.0).to(torch.int8))


@pytest.mark.gpu
def test_append_of_more_than_2_32_threads():
    """2^20 sequences of 256 kv heads: 2^28 warps, the last of which write the last sequences' rows."""
    from lara_b200 import kvquant, ops

    B, hkv, D = 2 ** 20, 256, 64
    starts, counts, table, some = _large_batch(B)
    pool = kvquant.QuantPool.empty(len(some), 16, hkv, D, "int8", DEV)
    rows = torch.randint(-127, 128, (hkv, 1, D), device=DEV)
    rows[..., 0] = 127
    x = rows.to(torch.bfloat16).expand(B, hkv, 1, D)
    new, st = torch.full_like(starts, -7), ops.new_workspace(256, DEV)
    kvquant.kvq_append(pool, table, starts, x, x, counts=counts, new_lens=new, workspace=st)
    assert ops.workspace_status(st) == 0
    assert torch.equal(new, starts + counts)
    for i, b in enumerate(some):
        for codes in (pool.k_codes, pool.v_codes):
            assert torch.equal(codes[i, :, int(starts[b])], rows[:, 0].to(torch.int8))
        assert torch.count_nonzero(pool.k_scales[i]) == hkv


@pytest.mark.gpu
def test_append_and_read_of_2_26_rows():
    """64 sequences of 8 kv heads padded to 131072 tokens, of which the last has any."""
    from lara_b200 import kvquant, ops

    B, hkv, n, D, ps = 64, 8, 131072, 64, 256
    table = torch.zeros((B, n // ps), dtype=torch.int32, device=DEV)
    table[-1] = torch.randperm(n // ps, device=DEV).to(torch.int32)
    pool = kvquant.QuantPool.empty(n // ps, ps, hkv, D, "int8", DEV)
    rows = torch.randint(-127, 128, (n, D), device=DEV)
    rows[:, 0] = 127
    x = rows.to(torch.bfloat16).expand(B, hkv, n, D)
    counts = torch.zeros(B, dtype=torch.int32, device=DEV)
    counts[-1] = n
    new, st = torch.full_like(counts, -7), ops.new_workspace(256, DEV)
    kvquant.kvq_append(pool, table, torch.zeros_like(counts), x, x, counts=counts, new_lens=new, workspace=st)
    assert torch.equal(new, counts)
    k, v = kvquant.kvq_read(pool, table, new, n, workspace=st)
    assert ops.workspace_status(st) == 0
    for y in (k, v):
        assert torch.equal(y[-1], x[-1]) and all(torch.count_nonzero(y[b]) == 0 for b in range(B - 1))


def test_rows_past_one_launch_are_refused():
    from test_kvquant import _append, _pool_struct, _read

    pool = _pool_struct()  # 2 kv heads, head_dim 128: a warp takes four tokens
    assert _append(pool, batch=1 << 12, n=1 << 20) == 0x01   # 2^31 warps
    assert _read(pool, batch=1 << 12, n=1 << 20) == 0x01
    assert _append(pool, batch=1 << 30, n=1) == 0x01
    assert _append(pool, batch=1, n=(1 << 30) + 1) == 0x01
    assert _append(pool, batch=0x7fffffff, n=0x7fffffff) == 0x01
    assert _append(pool, batch=1 << 30, n=0, k=None, v=None, new_lens=None) == 0


# ------------------------------------------------------------------ q/k head pass
def test_norm_rope_heads_past_31_bits_are_refused():
    """Products of the sizes that pass 64 bits among them (2^30 * 2^30 * 16 is 0 there)."""
    import ctypes

    from lara_b200._native import lib

    p, z = ctypes.c_void_p(4096), (0, 0, 0)
    for batch, n in ((1 << 30, 1 << 30), (1 << 16, 1 << 14), (0x7fffffff, 0x7fffffff), (1, 1 << 28)):
        assert lib.lara_qk_norm_rope(p, *z, p, *z, p, *z, p, *z, batch, n, 14, 2, 128, p, p, 16, 128, 1, p, p, 1e-5, None,
                                     None) == 0x01


# ------------------------------------------------------------------ decode: scales of V far from one another
def _page(rows, fmt):
    """rows [tokens, D] of one page of one kv head -> (codes, scales, values in 64 bits)."""
    from test_kvquant import DTYPES, quantise64, values64

    c, s = quantise64(rows, fmt)
    bits = c.to(torch.int8) if fmt == "int8" else c.float().to(torch.float8_e4m3fn)
    return bits.view(DTYPES[fmt]), s.float(), values64(c, s.float().double())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_many_tokens_without_values(fmt):
    """Hundreds of thousands of tokens whose V is zero, under rising scores, before as many whose V is one.

    The score is 0 for the first page and 7.9 octaves after it: the sum of weights is at its largest.
    """
    from lara_b200 import kvquant, ops

    B, D, ps, each = 64, 64, 256, 1536  # pages of zeros, pages of ones; every sequence has the same pages
    k, v = torch.zeros((3, ps, D)), torch.zeros((3, ps, D))
    k[1:, :, 0], v[2] = 1.0, 1.0
    pages = [[_page(x[i].to(torch.bfloat16), fmt) for i in range(3)] for x in (k, v)]
    codes = [torch.stack([p[0].view(torch.uint8) for p in q])[:, None].to(DEV).view(q[0][0].dtype) for q in pages]
    scales = [torch.stack([p[1] for p in q])[:, None].to(DEV) for q in pages]
    pool = kvquant.QuantPool(*codes, *scales)
    table = torch.tensor([0] + [1] * each + [2] * each, dtype=torch.int32, device=DEV).expand(B, -1).contiguous()
    lens = torch.full((B,), table.shape[1] * ps, dtype=torch.int32, device=DEV)
    q = torch.zeros((B, 2, D), dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 1.0
    ws = kvquant.decode_workspace(B, 2, 1, D, DEV)
    o = kvquant.gqa_decode_kvq(q, pool, table, lens, scale=7.9 * math.log(2.0), workspace=ws)
    assert ops.workspace_status(ws) == 0
    assert ((o.double() - each / (2 * each + 2.0 ** -7.9)).abs() <= 2.0 ** -8 * 0.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,G,D", [([768], 4, 64), ([512] * 1800, 2, 64), ([40000], 3, 128), ([4100] * 90, 9, 64)])
@pytest.mark.parametrize("large", [1e8, 1e20, 1e32])
def test_decode_zero_values_beside_large_ones(fmt, lens, G, D, large):
    """As many tokens of zeros as of large values, equally likely: in a warp's tiles, its neighbours', other CTAs'."""
    n = max(lens)
    g = torch.Generator().manual_seed(n)
    k, v = torch.zeros((1, n, D)), large * torch.randn((1, n, D), generator=g)
    k[:, :, 0], v[:, :n // 2] = 0.01 * torch.randn((1, n), generator=g), 0.0
    case = SharedRows(lens, 1, D, 64, fmt, k.to(torch.bfloat16), v.to(torch.bfloat16), seed=n)
    q = _rand_bf16(g, (len(lens), G, D), False).to(DEV)
    check_close(case, q, _decode_gpu(case, q), chain=384)


# ------------------------------------------------------------------ the one-launch step: padding
@pytest.mark.gpu
@pytest.mark.parametrize("given", [False, True])
def test_append_qkv_positions_of_padding_are_not_reported(given):
    """Ragged prompts padded past the rotation table; a counted row past it is reported."""
    from lara_b200 import kvquant, ops

    g = torch.Generator().manual_seed(3)
    B, n, hq, hkv, D, max_pos = 3, 200, 4, 2, 64, 1000
    x = _rand_bf16(g, (B, n, hq + 2 * hkv, D)).to(DEV)
    args = (x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:])
    table = torch.arange(3 * 20, dtype=torch.int32, device=DEV).view(3, 20)
    pool = kvquant.QuantPool.empty(60, 64, hkv, D, "int8", DEV)
    tab = ops.rope_table(max_pos, D, device=DEV)
    starts = _i32([900, 0, 999])
    pos = (starts[:, None] + torch.arange(n, dtype=torch.int32, device=DEV)) if given else None
    if given:
        pos[1, 150:] = -5
    st, new = ops.new_workspace(256, DEV), _i32([0] * 3)
    for counts, bits in (([100, 150, 1], 0), ([0, 0, 0], 0), ([101, 1, 1], 0x10), ([1, 1, 2], 0x10), ([-1, 201, 1], 0x2)):
        if given and counts[1] > 150:
            bits |= 0x10
        kvquant.kvq_append_qkv(pool, table, starts, *args, positions=pos, cos_sin=tab, counts=_i32(counts), new_lens=new,
                               workspace=st)
        assert ops.workspace_status(st) == bits, counts
        assert new.tolist() == [s + min(max(c, 0), n) for s, c in zip((900, 0, 999), counts)]


# ------------------------------------------------------------------ decode: workspaces
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_workspace_of_other_calls(fmt):
    """One workspace, made for the most heads: every geometry, batch and way of joining after every other."""
    from lara_b200 import kvquant, ops

    g = torch.Generator().manual_seed(17)
    cases = []
    for lens, hkv, G, D in (([2000] * 70, 2, 16, 128), ([9000, 20], 1, 16, 128), ([6000], 2, 4, 64),
                            ([2000] * 70, 2, 1, 128), ([30000], 1, 5, 64), ([700] * 200, 4, 12, 64),
                            ([300], 8, 4, 128), ([40000], 1, 3, 128)):
        rows = [_rand_bf16(g, (hkv, max(lens), D)) for _ in range(2)]
        case = SharedRows(lens, hkv, D, 64, fmt, *rows, seed=len(lens))
        q = _rand_bf16(g, (len(lens), hkv * G, D), False).to(DEV)
        cases.append((case, q, _decode_gpu(case, q)))
    ws = kvquant.decode_workspace(1, 16, 1, 128, DEV)
    for i in torch.randperm(4 * len(cases), generator=g).tolist():
        case, q, want = cases[i % len(cases)]
        own = q.clone()
        for query, out in ((q, torch.full_like(q, 3.0)), (own, own)):  # into another tensor, and into the queries
            kvquant.gqa_decode_kvq(query, case.pool, case.dtable, case.dlens, workspace=ws, out=out)
            assert torch.equal(out, want), i % len(cases)
    assert ops.workspace_status(ws) == 0


def test_decode_workspace_bytes_do_not_depend_on_the_batch():
    from lara_b200._native import lib

    b = lib.lara_kvq_decode_workspace_bytes
    assert b(1, 32, 8, 128) == b(4096, 32, 8, 128) == b(7, 4, 1, 128) > b(1, 8, 8, 128) > 0


# ------------------------------------------------------------------ sizes past 32 bits in Python's calls
@pytest.mark.gpu
def test_sizes_past_32_bits_are_refused():
    """2^32 + 128 must not be taken for 128; the tensors are empty and take no memory."""
    from lara_b200 import kvquant, ops

    big = (1 << 32) + 128
    pool = kvquant.QuantPool.empty(2, 16, 1, 64, "int8", DEV)
    none = torch.empty((0,), dtype=torch.int32, device=DEV)
    rows = torch.empty((0, 1, 1, 64), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="pages per sequence is too large"):
        kvquant.kvq_append(pool, torch.empty((0, big), dtype=torch.int32, device=DEV), none, rows, rows)
    x = torch.empty((0, 1, big), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="head_dim is too large"):
        ops.qk_norm_rope(x, x, cos_sin=torch.empty((4, 64), device=DEV), positions=none)
    x = torch.empty((0, 1, 64), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="rot_dim is too large"):
        ops.qk_norm_rope(x, x, cos_sin=torch.empty((0, big), device=DEV), positions=none)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 127, 128, 129, 5000])
def test_append_lengths_without_rows(B):
    """n = 0: the lengths of every sequence, by as many blocks as they need."""
    from lara_b200 import kvquant

    pool = kvquant.QuantPool.empty(1, 16, 1, 64, "int8", DEV)
    table = torch.zeros((B, 1), dtype=torch.int32, device=DEV)
    starts = torch.arange(B, dtype=torch.int32, device=DEV) % 17
    none = torch.empty((B, 1, 0, 64), dtype=torch.bfloat16, device=DEV)
    new = torch.full_like(starts, -7)
    kvquant.kvq_append(pool, table, starts, none, none, new_lens=new)
    assert torch.equal(new, starts)
    new.fill_(-7)
    heads = none.transpose(1, 2)
    kvquant.kvq_append_qkv(pool, table, starts, heads, heads, heads, new_lens=new)
    assert torch.equal(new, starts)
