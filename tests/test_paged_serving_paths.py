"""Paths of the paged cache's serving operators that short calls do not take, each against its definition in 64 bits.

Tolerances are those of ``test_paged_serving``.
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from test_paged_serving import check_out, check_weights, decode64, dev, make_cache, rows64, words  # noqa: E402


# ------------------------------------------------------------------ scores of minus infinity
def masked64(q, k, v, table, lens, page, scale, masked):
    """:func:`decode64` where the tokens of ``masked[b]`` have scores of -inf; rows that have no others give zeros."""
    B, hq, d = q.shape
    hkv = k.shape[1]
    o = torch.zeros((B, hq, d), dtype=torch.float64)
    kappa, A, ps = torch.zeros_like(o), torch.zeros((B, hq, 1), dtype=torch.float64), []
    for b in range(B):
        n = int(lens[b])
        ks, vs = (rows64(x, table, b, n, page).transpose(0, 1) for x in (k, v))
        off = torch.zeros(n, dtype=torch.bool)
        off[torch.tensor(masked[b], dtype=torch.long)] = True
        ks = ks.masked_fill(off[None, :, None], 0.0)
        qs = q[b].double().view(hkv, -1, d)
        p = torch.softmax((qs @ ks.transpose(1, 2) * scale).masked_fill(off, -math.inf), -1).nan_to_num(0.0)
        ps.append(p)
        o[b] = (p @ vs).view(hq, d)
        kappa[b] = (p @ vs.abs()).view(hq, d)
        A[b] = ((qs.abs() @ ks.abs().transpose(1, 2)) * scale).amax(-1).view(hq, 1)
    return o, kappa, A, ps


def mask_tokens(k, table, page, masked, word):
    """Keys whose products with queries of 8 in the first two places are -inf (in fp32, where ``word`` is finite)."""
    for b, ts in enumerate(masked):
        for t in ts:
            k[int(table[b, t // page]), :, t % page, :2] = word


LOWEST = -3.3895e38  # of bf16: 8 times it is -inf in fp32


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (10, 2, 64), (32, 2, 128)])
@pytest.mark.parametrize("word", [-math.inf, LOWEST])
def test_scored_decode_of_scores_of_minus_infinity(hq, hkv, d, word):
    """Pages of keys that mask, first, in the middle and last; the last sequence has no other tokens."""
    from lara_b200 import ops, paged

    page, lens = 16, [400, 1000, 37, 400, 48]
    k, v, table, n = make_cache(lens, hkv, d, page, seed=d + hq)
    masked = [range(16), range(320, 352), range(32, 37), [t for t in range(400) if t // 16 % 3 != 1], range(48)]
    mask_tokens(k, table, page, masked, word)
    g = torch.Generator().manual_seed(31)
    q = torch.randn((len(lens), hq, d), generator=g).bfloat16()
    q[..., :2] = 8.0
    w = torch.rand(k.shape[:3], generator=g)
    o, kappa, A, ps = masked64(q, k, v, table, n, page, d ** -0.5, masked)
    qd, kd, vd, wd, td, nd = dev(q, k, v, w, table, n)
    ws = paged.scored_workspace(len(lens), hq, kd, table.shape[1])
    check_out(paged.gqa_decode_scored(qd, kd, vd, wd, td, nd, workspace=ws), o, kappa, A, n)
    check_weights(wd, w, ps, A, table, n, page, d)
    assert ops.workspace_status(ws) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,batch", [(8, 2, 128, 3), (10, 2, 64, 3), (32, 2, 128, 20), (16, 2, 64, 40)])
@pytest.mark.parametrize("word", [-math.inf, LOWEST])
@pytest.mark.parametrize("where", ["first", "middle", "last", "all", "own"])
def test_shared_decode_of_scores_of_minus_infinity(hq, hkv, d, batch, word, where):
    """Keys that mask in the prefix (in tiles of 128 tokens, whole and half) or in the own tokens; one sequence without
    own tokens, which has nothing to attend where the whole prefix masks."""
    from lara_b200 import ops, paged

    page, shared = 64, 8
    prefix = shared * page
    lens = [prefix + 50] * batch
    lens[1], lens[2] = prefix, 300  # at the prefix's end, and within it, of pages that it has in common
    k, v, table, n = make_cache(lens, hkv, d, page, seed=d + hq, shared=shared)
    tokens = {"first": range(192), "middle": range(128, 320), "last": range(prefix - 192, prefix),
              "all": range(prefix), "own": range(prefix, prefix + 50)}[where]
    masked = [[t for t in tokens if t < m] for m in lens]
    mask_tokens(k, table, page, masked, word)
    q = torch.randn((batch, hq, d), generator=torch.Generator().manual_seed(32)).bfloat16()
    q[..., :2] = 8.0
    o, kappa, A, _ = masked64(q, k, v, table, n, page, d ** -0.5, masked)
    qd, kd, vd, td, nd = dev(q, k, v, table, n)
    ws = paged.shared_workspace(batch, hq, hkv, d, "cuda")
    for front in (shared, 0):  # and every sequence for itself
        check_out(paged.gqa_decode_shared(qd, kd, vd, td, nd, front, workspace=ws), o, kappa, A, n)
    assert ops.workspace_status(ws) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,batch", [(8, 2, 128, 3), (10, 2, 64, 3), (32, 2, 128, 20), (16, 2, 64, 40)])
@pytest.mark.parametrize("size", [2.0 ** -6, 0.5, 1.0])
@pytest.mark.parametrize("where", ["first", "middle", "last", "all", "own"])
def test_decodes_of_finite_scores_that_mask(hq, hkv, d, batch, size, where):
    """Keys of the type's lowest value whose scores are finite, -10^35 to -10^38: they weigh nothing beside others."""
    from lara_b200 import paged

    page, shared = 64, 8
    prefix = shared * page
    lens = [prefix + 50 + b % 7 for b in range(batch)]
    k, v, table, n = make_cache(lens, hkv, d, page, seed=d + hq, shared=shared)
    tokens = {"first": range(192), "middle": range(128, 320), "last": range(prefix - 192, prefix),
              "all": range(prefix), "own": range(prefix, prefix + 50 - 13)}[where]
    masked = [list(tokens)] * batch
    mask_tokens(k, table, page, masked, LOWEST)
    q = torch.randn((batch, hq, d), generator=torch.Generator().manual_seed(34)).bfloat16()
    q[..., :2] = size
    o, kappa, A, _ = masked64(q, k, v, table, n, page, d ** -0.5, masked)
    qd, kd, vd, td, nd = dev(q, k, v, table, n)
    for front in (shared, 0):
        check_out(paged.gqa_decode_shared(qd, kd, vd, td, nd, front), o, kappa, A, n)
    if batch == 3:  # a sequence of its own, scored
        w = torch.zeros(k.shape[:3])
        o, kappa, A, ps = masked64(q[:1], k, v, table[:1], n[:1], page, d ** -0.5, masked[:1])
        wd = w.cuda()
        check_out(paged.gqa_decode_scored(qd[:1], kd, vd, wd, td[:1], nd[:1]), o, kappa, A, n[:1])
        check_weights(wd, w, ps, A, table[:1], n[:1], page, d)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,batch", [(8, 2, 128, 3), (10, 2, 64, 3), (16, 2, 64, 40)])
@pytest.mark.parametrize("size", [2.0 ** -96, 2.0 ** -6, 0.5])
def test_decodes_of_one_score_above_all(hq, hkv, d, batch, size):
    """A finite score of 10^9 to 10^38 takes all the weight, wherever it is: the output is that token's value."""
    from lara_b200 import paged

    page, shared = 64, 8
    prefix = shared * page
    lens = [prefix + 50] * batch
    for at in (0, 200, prefix - 1, prefix + 20):
        k, v, table, n = make_cache(lens, hkv, d, page, seed=d + hq, shared=shared)
        mask_tokens(k, table, page, [[at]] * batch, -LOWEST)
        q = torch.randn((batch, hq, d), generator=torch.Generator().manual_seed(35)).bfloat16()
        q[..., :2] = size
        qd, kd, vd, td, nd = dev(q, k, v, table, n)
        for front in (shared, 0):
            got = paged.gqa_decode_shared(qd, kd, vd, td, nd, front).cpu().view(batch, hkv, -1, d)
            for b in range(batch):
                want = v[int(table[b, at // page]), :, at % page]
                assert torch.equal(got[b], want[:, None].expand_as(got[b]))


# ------------------------------------------------------------------ long prefixes
@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,batch,page,shared", [
    (32, 8, 128, 4, 256, 160),   # one row tile, 320 token tiles to a kv head: runs that cross kv heads in mid-prefix
    (28, 4, 64, 3, 16, 2507),    # the same of pages smaller than a tile, the last tile in part
    (8, 2, 128, 70, 64, 315),    # row tiles: one pair and one alone
    (64, 4, 64, 30, 128, 157),   # groups of 16, four row tiles
    (6, 1, 128, 150, 32, 1001)])
def test_shared_decode_behind_a_long_prefix(hq, hkv, d, batch, page, shared):
    """Many token tiles for each CTA, and scores that grow along the prefix, so that references move late."""
    from lara_b200 import ops, paged

    prefix = shared * page
    lens = [prefix + (7 * b) % 90 for b in range(batch)]
    lens[1] = prefix - 3
    k, v, table, n = make_cache(lens, hkv, d, page, seed=hq + batch, shared=shared)
    grow = (1.0 + 2.0 * torch.arange(shared) / shared).view(-1, 1, 1, 1)
    at = table[0, :shared].long()
    k[at] = (k[at].float() * grow).bfloat16()
    q = torch.randn((batch, hq, d), generator=torch.Generator().manual_seed(33)).bfloat16()
    qd, kd, vd, td, nd = dev(q, k, v, table, n)
    o, kappa, A, _ = decode64(qd, kd, vd, td, nd, page, d ** -0.5)
    ws = paged.shared_workspace(batch, hq, hkv, d, "cuda")
    got = paged.gqa_decode_shared(qd, kd, vd, td, nd, shared, workspace=ws)
    check_out(got, o, kappa, A, n)
    assert torch.equal(words(paged.gqa_decode_shared(qd, kd, vd, td, nd, shared, workspace=ws)), words(got))
    assert ops.workspace_status(ws) == 0


# ------------------------------------------------------------------ long evictions
@pytest.mark.gpu
@pytest.mark.parametrize("lens,page,keep,hkv", [
    ([700000], 64, 100003, 1),          # more keys to a CTA than its shared memory holds
    ([640000, 13, 520001], 16, 300007, 1),  # and more table entries
    ([1 << 20], 256, 1000, 2), ([600000], 16, 599999, 1)])
@pytest.mark.parametrize("kind", ["many", "ties"])
def test_evict_of_very_long_sequences(lens, page, keep, hkv, kind):
    from lara_b200 import ops, paged

    d = 64
    used = [-(-m // page) for m in lens]
    g = torch.Generator(device="cuda").manual_seed(len(lens) + keep)
    order = torch.randperm(sum(used) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(used) + 1), -1, dtype=torch.int32, device="cuda")
    for b, u in enumerate(used):
        table[b, :u] = order[sum(used[:b]):sum(used[:b + 1])]
    shape = (sum(used) + 3, hkv, page)
    k, v = (torch.randint(-32768, 32768, (*shape, d), generator=g, device="cuda", dtype=torch.int16) for _ in "kv")
    w = torch.randint(0, 3 if kind == "ties" else 1 << 22, shape, generator=g, device="cuda").float() / 64
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    src = torch.empty((len(lens), hkv, keep), dtype=torch.int32, device="cuda")
    ws = paged.evict_workspace(len(lens), hkv, keep, "cuda")
    new = paged.kv_evict(k, v, w, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), keep, first=3, last=77,
                         sources=src, workspace=ws)
    assert new.tolist() == [min(m, keep) for m in lens]
    free = torch.ones(shape[0], dtype=torch.bool, device="cuda")
    for b, m in enumerate(lens):
        t = torch.arange(m, device="cuda")
        pages, rows = table[b].long()[t // page], t % page
        free[pages] = False
        for h in range(hkv):
            at = (pages, h, rows)
            want = torch.arange(keep, device="cuda")
            if m <= keep:
                want[m:] = -1
                assert torch.equal(src[b, h].long(), want)
                assert torch.equal(k[at], k0[at]) and torch.equal(v[at], v0[at]) and torch.equal(w[at], w0[at])
                continue
            x = w0[at].clone()
            x[:3] = x[m - 77:] = math.inf
            kept = torch.zeros(m, dtype=torch.bool, device="cuda")
            kept[torch.sort(x, descending=True, stable=True).indices[:keep]] = True
            want[~kept[:keep]] = torch.nonzero(kept[keep:]).flatten() + keep
            assert torch.equal(src[b, h].long(), want)
            assert torch.equal(w[at][:keep], w0[at][want]) and not w[at][keep:].any()
            assert torch.equal(k[at][:keep], k0[at][want]) and torch.equal(v[at][:keep], v0[at][want])
            assert torch.equal(k[at][keep:], k0[at][keep:])
    assert torch.equal(w[free], w0[free]) and torch.equal(k[free], k0[free])
    assert ops.workspace_status(ws) == 0
