"""Serving operators of the paged bf16 cache (``lara_b200.paged``): the decode behind a shared prefix, the decode that
scores its cache, and eviction by gathered weight.

Each is compared with its definition in 64 bits.  Tolerances:

* decode, one bf16 rounding of the result (2^-8 of it), and relative to ``kappa = sum_t p_t |v_t|``: weights held in
  two bf16 numbers (2^-8 of 2^-8), the exponential and its products (2^-21), the score in fp32 (D + 8 roundings of at
  most 2^-23 of ``A = max_t scale sum_d |q_d k_td|``, above and below the line), and sums over n tokens (n 2^-22: a
  tensor core may cut where it adds);
* weights: the same without V, and one fp32 rounding of each of the sum's terms (2^-23);
* eviction moves words and is exact.
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

GEOMETRIES = [(1, 1, 128), (4, 1, 64), (8, 2, 128), (10, 2, 64), (21, 3, 128), (16, 2, 128), (15, 1, 64), (32, 2, 128)]


# ------------------------------------------------------------------ inputs
def make_cache(lens, hkv, d, page, seed, shared=0, spare=0):
    """Pools with a NaN in every row that no sequence has, a table of pages in random order; all on the CPU."""
    g = torch.Generator().manual_seed(seed)
    per_seq = max(1, -(-max(lens) // page)) + spare
    used = [max(0, -(-n // page) - shared) for n in lens]
    pages = shared + sum(used) + 2
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), per_seq), -1, dtype=torch.int32)
    table[:, :shared] = order[:shared]
    at = shared
    for b, u in enumerate(used):
        table[b, shared:shared + u] = order[at:at + u]
        at += u
    k = torch.randn((pages, hkv, page, d), generator=g)
    k[..., 1::d // 4] *= 6.0
    v = torch.randn((pages, hkv, page, d), generator=g)
    there = torch.zeros((pages, page), dtype=torch.bool)
    for b, n in enumerate(lens):
        t = torch.arange(n)
        there[table[b].long()[t // page], t % page] = True
    for x in (k, v):
        x.masked_fill_(~there[:, None, :, None], math.nan)
    return k.bfloat16(), v.bfloat16(), table, torch.tensor(lens, dtype=torch.int32)


def rows64(x, table, b, n, page):
    t = torch.arange(n)
    return x[table[b].long()[t // page], :, t % page].double()  # [n, hkv, d]


def decode64(q, k, v, table, lens, page, scale):
    """o, kappa, A [B, Hq, D or 1], and the weights p [B][hkv, G, n]."""
    B, hq, d = q.shape
    hkv = k.shape[1]
    o = torch.zeros((B, hq, d), dtype=torch.float64)
    kappa, A, ps = torch.zeros_like(o), torch.zeros((B, hq, 1), dtype=torch.float64), []
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            ps.append(None)
            continue
        ks, vs = (rows64(x, table, b, n, page).transpose(0, 1) for x in (k, v))
        qs = q[b].double().view(hkv, -1, d)
        p = torch.softmax(qs @ ks.transpose(1, 2) * scale, -1)
        ps.append(p)
        o[b] = (p @ vs).view(hq, d)
        kappa[b] = (p @ vs.abs()).view(hq, d)
        A[b] = ((qs.abs() @ ks.abs().transpose(1, 2)) * scale).amax(-1).view(hq, 1)
    return o, kappa, A, ps


def relative(A, d, n):
    return 2.0 ** -16 + 2.0 ** -21 + 2 * (d + 8) * 2.0 ** -23 * A + n * 2.0 ** -22


def check_out(got, o, kappa, A, lens):
    n = lens.double().view(-1, 1, 1)
    tol = 2.0 ** -8 * o.abs() + kappa * relative(A, o.shape[-1], n)
    err = (got.cpu().double() - o).abs()
    assert torch.isfinite(got.float()).all()
    assert (err <= tol).all(), f"{float((err - tol).max())} over the tolerance, {int((err > tol).sum())} values"


def check_weights(got, before, ps, A, table, lens, page, d):
    want, tol = before.double().clone(), 2.0 ** -23 * before.double().abs()
    touched = torch.zeros(before.shape, dtype=torch.bool)
    for b, p in enumerate(ps):
        if p is None:
            continue
        n, (hkv, G) = p.shape[2], p.shape[:2]
        rel = relative(A[b].view(hkv, G, 1), d, n) + G * 2.0 ** -23
        t = torch.arange(n)
        at = (table[b].long()[t // page], slice(None), t % page)
        want[at] += p.sum(1).t()
        tol[at] += (p * rel).sum(1).t() + 2.0 ** -23 * want[at].abs()
        touched[at] = True
    got = got.cpu()
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"{float((err - tol).max())} over the tolerance"
    assert torch.equal(got[~touched], before[~touched])


def evict64(k, v, w, table, lens, page, keep, first, last):
    """The definition, slot by slot: new k, v, w, sources, lengths."""
    k, v, w = k.clone(), v.clone(), w.clone()
    B, hkv = len(lens), k.shape[1]
    src = torch.full((B, hkv, keep), -1, dtype=torch.int32)
    for b in range(B):
        n = int(lens[b])
        page_of = [int(x) for x in table[b]]
        for h in range(hkv):
            if n <= keep:
                src[b, h, :n] = torch.arange(n)
                continue
            at = [(page_of[t // page], h, t % page) for t in range(n)]
            ws = [float(w[x]) for x in at]
            heavy = lambda t: (math.inf if math.isnan(ws[t]) else ws[t], math.isnan(ws[t]))  # noqa: E731
            middle = sorted(range(first, n - last), key=lambda t: (heavy(t), -t), reverse=True)
            kept = set(range(first)) | set(range(n - last, n)) | set(middle[:keep - first - last])
            holes = [t for t in range(keep) if t not in kept]
            movers = sorted(t for t in kept if t >= keep)
            assert len(holes) == len(movers)
            src[b, h] = torch.arange(keep)
            for t, s in zip(holes, movers):
                k[at[t]], v[at[t]], w[at[t]] = k[at[s]], v[at[s]], w[at[s]]
                src[b, h, t] = s
            for t in range(keep, n):
                w[at[t]] = 0.0
    return k, v, w, src, torch.clamp(lens, max=keep)


def words(x):
    return x.cpu().contiguous().view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32)


def dev(*xs):
    return [x.cuda() for x in xs]


# ------------------------------------------------------------------ decode with scores
@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", GEOMETRIES)
@pytest.mark.parametrize("page,lens", [(16, [1]), (16, [17, 0, 1, 16, 300, 33]), (64, [1000, 0, 63, 64, 65]),
                                       (256, [5000])])
def test_scored_decode(hq, hkv, d, page, lens):
    from lara_b200 import ops, paged

    k, v, table, n = make_cache(lens, hkv, d, page, seed=hq * 7 + d + page, spare=2)
    g = torch.Generator().manual_seed(5)
    q = torch.randn((len(lens), hq, d), generator=g).bfloat16()
    w = torch.rand(k.shape[:3], generator=g)
    scale = 1.0 / math.sqrt(d)
    o, kappa, A, ps = decode64(q, k, v, table, n, page, scale)
    qd, kd, vd, wd, td, nd = dev(q, k, v, w, table, n)
    ws = paged.scored_workspace(len(lens), hq, kd, table.shape[1])
    apart = torch.full_like(wd, -7.0)
    for _ in range(2):  # the weights apart from the old ones, twice, then in place
        got = paged.gqa_decode_scored(qd, kd, vd, wd, td, nd, weights_out=apart, workspace=ws)
        check_out(got, o, kappa, A, n)
    again = paged.gqa_decode_scored(qd, kd, vd, wd, td, nd)
    assert torch.equal(words(again), words(got))
    check_weights(wd, w, ps, A, table, n, page, d)
    there = apart != -7.0
    assert torch.equal(apart[there], wd[there])
    assert torch.equal(wd.cpu()[~there.cpu()], w[~there.cpu()])
    assert ops.workspace_status(ws) == 0


# ------------------------------------------------------------------ decode behind a shared prefix
@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", GEOMETRIES)
@pytest.mark.parametrize("page,shared,lens", [
    (16, 1, [17, 16, 40]), (16, 9, [150, 144, 145, 0, 143, 16, 1]), (64, 5, [400, 321, 320, 100]),
    (16, 63, [1009] * 40 + [1008, 5]), (256, 4, [1300, 1024]), (32, 0, [70, 3]), (32, 4, [128] * 3)])
def test_shared_decode(hq, hkv, d, page, shared, lens):
    from lara_b200 import ops, paged

    k, v, table, n = make_cache(lens, hkv, d, page, seed=hq + d + page + shared, shared=shared)
    q = torch.randn((len(lens), hq, d), generator=torch.Generator().manual_seed(9)).bfloat16()
    o, kappa, A, _ = decode64(q, k, v, table, n, page, 0.11)
    qd, kd, vd, td, nd = dev(q, k, v, table, n)
    ws = paged.shared_workspace(len(lens), hq, hkv, d, "cuda")
    got = paged.gqa_decode_shared(qd, kd, vd, td, nd, shared, scale=0.11, workspace=ws)
    check_out(got, o, kappa, A, n)
    assert torch.equal(words(paged.gqa_decode_shared(qd, kd, vd, td, nd, shared, scale=0.11, workspace=ws)), words(got))
    out = qd.clone()
    paged.gqa_decode_shared(out, kd, vd, td, nd, shared, scale=0.11, workspace=ws, out=out)
    assert torch.equal(words(out), words(got))
    assert ops.workspace_status(ws) == 0


# ------------------------------------------------------------------ eviction
@pytest.mark.gpu
@pytest.mark.parametrize("page,lens,keep,first,last", [
    (16, [2], 1, 0, 0), (16, [40, 0, 17, 16, 15, 1], 16, 0, 0), (16, [40, 33, 300], 32, 32, 0),
    (16, [40, 33, 300], 32, 0, 32), (64, [1000, 513, 700], 512, 4, 100), (256, [3000], 700, 3, 7),
    (16, [500, 90], 100, 30, 70), (16, [64, 10], 640, 1, 1), (32, [9000], 8999, 2, 2), (32, [9000], 1, 0, 0)])
@pytest.mark.parametrize("hkv,d", [(1, 64), (3, 128)])
@pytest.mark.parametrize("kind", ["any", "ties", "special"])
def test_evict(page, lens, keep, first, last, hkv, d, kind):
    from lara_b200 import ops, paged

    k, v, table, n = make_cache(lens, hkv, d, page, seed=keep + d, spare=1)
    g = torch.Generator().manual_seed(3)
    w = torch.exp(torch.randn(k.shape[:3], generator=g) * 3)
    if kind == "ties":
        w = torch.randint(0, 4, w.shape, generator=g).float()
    if kind == "special":
        pick = torch.randint(0, 9, w.shape, generator=g)
        for i, x in enumerate((math.inf, -math.inf, math.nan, 0.0, -0.0, 1e-42, -1e-42)):
            w[pick == i] = x
        w[pick == 7] *= -1.0
    want = evict64(k, v, w, table, n, page, keep, first, last)
    for apart in (False, True):
        kd, vd, wd, td, nd = dev(k, v, w, table, n)
        w_out = wd.clone() if apart else wd
        src = torch.full((len(lens), hkv, keep), 99, dtype=torch.int32, device="cuda")
        ws = paged.evict_workspace(len(lens), hkv, keep, "cuda")
        new = paged.kv_evict(kd, vd, wd, td, nd, keep, first=first, last=last, weights_out=w_out, sources=src,
                             workspace=ws)
        assert torch.equal(new.cpu(), want[4]) and torch.equal(nd.cpu(), n)
        assert torch.equal(src.cpu(), want[3])
        for got, x in zip((kd, vd, w_out), want):
            assert torch.equal(words(got), words(x))
        if apart:
            assert torch.equal(words(wd), words(w))
        assert ops.workspace_status(ws) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("lens,keep", [([70000, 5, 40001], 1003), ([300000], 150001)])
def test_evict_long(lens, keep):
    """Units that a cluster of CTAs selects from, against a sort."""
    from lara_b200 import paged

    hkv, d, page = 2, 64, 64
    k, v, table, n = make_cache(lens, hkv, d, page, seed=1)
    w = torch.randint(0, 5000, k.shape[:3], generator=torch.Generator().manual_seed(2)).float() / 64
    kd, vd, wd, td, nd = dev(k, v, w, table, n)
    src = torch.empty((len(lens), hkv, keep), dtype=torch.int32, device="cuda")
    paged.kv_evict(kd, vd, wd, td, nd, keep, first=3, last=77, sources=src)
    src, w_new = src.cpu(), wd.cpu()
    for b, m in enumerate(lens):
        t = torch.arange(m)
        at = (table[b].long()[t // page], t % page)
        for h in range(hkv):
            if m <= keep:
                assert src[b, h].tolist() == list(range(m)) + [-1] * (keep - m)
                continue
            x = w[at[0], h, at[1]]
            x[:3] = x[m - 77:] = math.inf
            kept = torch.zeros(m, dtype=torch.bool)
            kept[torch.sort(x, descending=True, stable=True).indices[:keep]] = True
            want = torch.arange(keep)
            want[~kept[:keep]] = torch.nonzero(kept[keep:]).flatten() + keep
            assert torch.equal(src[b, h].long(), want)
            now = w_new[at[0], h, at[1]]
            assert torch.equal(now[:keep], w[at[0], h, at[1]][want]) and not now[keep:].any()
            for new, old in ((kd, k), (vd, v)):
                assert torch.equal(words(new[:, h].cpu()[at[0], at[1]][:keep]), words(old[at[0], h, at[1]][want]))


# ------------------------------------------------------------------ the cache's methods, together
@pytest.mark.gpu
def test_serving_loop():
    """Prompts behind a shared prefix decode; then scored steps, evictions and appends, against a model on the CPU."""
    from lara_b200.paged import PagedKVCache

    hq, hkv, d, page = 8, 2, 64, 16
    g = torch.Generator().manual_seed(11)
    rows = lambda n: torch.randn((1, hkv, n, d), generator=g).bfloat16()  # noqa: E731
    cache = PagedKVCache(64, page, hkv, d, 4, 320, "cuda")
    cache.new_sequence()
    doc = rows(70), rows(70)
    cache.append(doc[0].cuda(), doc[1].cuda(), [0])
    own = {}
    for s in (1, 2):
        assert cache.new_sequence() == s
        assert cache.share_prefix(0, s, 70) == 64
        own[s] = rows(s * 9), rows(s * 9)
        cache.append(own[s][0].cuda(), own[s][1].cuda(), [s])
    assert cache.shared_pages() == 4
    q = torch.randn((3, hq, d), generator=g).bfloat16()
    got = cache.decode_shared(q.cuda())
    lens = torch.tensor([70, 73, 82])
    args = decode64(q, cache.k_pages.cpu(), cache.v_pages.cpu(), cache.block_table.cpu(), lens, page, d ** -0.5)
    check_out(got, *args[:3], lens)
    assert cache.status() == 0

    cache = PagedKVCache(24, page, hkv, d, 2, 160, "cuda", scored=True)
    have = {}
    for s, n in ((0, 100), (1, 31)):
        assert cache.new_sequence() == s
        x = rows(n), rows(n)
        cache.append(x[0].cuda(), x[1].cuda(), [s])
        have[s] = n
    for step in range(40):
        new = torch.randn((2, hkv, 1, d), generator=g).bfloat16(), torch.randn((2, hkv, 1, d), generator=g).bfloat16()
        cache.append(new[0].cuda(), new[1].cuda())
        have = {s: n + 1 for s, n in have.items()}
        before = cache.weights.cpu()
        q = torch.randn((2, hq, d), generator=g).bfloat16()
        got = cache.decode_scored(q.cuda())
        lens = torch.tensor([have[0], have[1]], dtype=torch.int32)
        table = cache.block_table.cpu()
        args = decode64(q, cache.k_pages.cpu(), cache.v_pages.cpu(), table, lens, page, d ** -0.5)
        check_out(got, *args[:3], lens)
        check_weights(cache.weights, before, args[3], args[2], table, lens, page, d)
        if step % 5 == 4:
            state = [x.cpu() for x in (cache.k_pages, cache.v_pages, cache.weights)]
            want = evict64(*state, table, lens, page, 48, 2, 5)
            src = torch.empty((2, hkv, 48), dtype=torch.int32, device="cuda")
            cache.evict(48, first=2, last=5, sources=src)
            have = {s: min(n, 48) for s, n in have.items()}
            for x, y in zip((cache.k_pages, cache.v_pages, cache.weights, src, cache.lens), want):
                assert torch.equal(words(x), words(y))
            assert [cache.seq_len(s) for s in (0, 1)] == [have[0], have[1]]
            assert cache.free_pages == 24 - sum(-(-n // page) for n in have.values())
    assert cache.status() == 0


# ------------------------------------------------------------------ what else a call may meet
@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (10, 2, 64)])
def test_shared_decode_of_a_padded_batch(hq, hkv, d):
    """Rows that do not cover the prefix need not name it: padding without pages, a short sequence with its own."""
    from lara_b200 import ops, paged

    page, shared, lens = 32, 3, [0, 40, 96, 200, 0, 97]
    k, v, table, n = make_cache(lens, hkv, d, page, seed=2, shared=shared, spare=1)
    used = set(table.flatten().tolist())
    own = torch.tensor([[x for x in range(k.shape[0]) if x not in used]])  # two pages, of no sequence
    g = torch.Generator().manual_seed(8)
    for x in (k, v):
        x[own[0]] = torch.randn(x[own[0]].shape, generator=g).bfloat16()
        x[own[0, 1], :, 8:] = math.nan
    table[0], table[4], table[1] = -1, 1 << 30, -7
    table[1, :2] = own[0].int()
    q = torch.randn((len(lens), hq, d), generator=g).bfloat16()
    o, kappa, A, _ = decode64(q, k, v, table, n, page, d ** -0.5)
    qd, kd, vd, td, nd = dev(q, k, v, table, n)
    ws = paged.shared_workspace(len(lens), hq, hkv, d, "cuda")
    check_out(paged.gqa_decode_shared(qd, kd, vd, td, nd, shared, workspace=ws), o, kappa, A, n)
    assert ops.workspace_status(ws) == 0
    # no sequence covers it: nothing of it is read
    table[:, 2:] = -1
    n = torch.minimum(n, torch.tensor(64, dtype=torch.int32))
    o, kappa, A, _ = decode64(q, k, v, table, n, page, d ** -0.5)
    check_out(paged.gqa_decode_shared(qd, kd, vd, table.cuda(), n.cuda(), shared, workspace=ws), o, kappa, A, n)
    assert ops.workspace_status(ws) == 0


@pytest.mark.gpu
def test_lengths_and_pages_out_of_range():
    """Lengths are clamped and bad pages not written; both are flagged."""
    from lara_b200 import ops, paged

    hq, hkv, d, page = 8, 2, 64, 16
    k, v, table, n = make_cache([40, 64, 20], hkv, d, page, seed=4)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    w = torch.rand(k.shape[:3])
    q = torch.randn((3, hq, d)).bfloat16()
    table[0, 1] = k.shape[0]
    raw = torch.tensor([40, 70, -3], dtype=torch.int32)  # past the capacity of 64, below 0
    qd, kd, vd, wd, td, nd = dev(q, k, v, w, table, raw)
    want = torch.tensor([40, 64, 0], dtype=torch.int32)
    seen = table.clone()
    seen[0, 1] = 0  # page 0 is read in its place
    o, kappa, A, _ = decode64(q, k, v, seen, want, page, 0.125)
    ws = paged.scored_workspace(3, hq, kd, table.shape[1])
    check_out(paged.gqa_decode_scored(qd, kd, vd, wd, td, nd, scale=0.125, workspace=ws), o, kappa, A, want)
    assert ops.workspace_status(ws) == 2 + 8 and ops.workspace_status(ws) == 0
    ws = paged.shared_workspace(3, hq, hkv, d, "cuda")
    check_out(paged.gqa_decode_shared(qd, kd, vd, td, nd, 0, scale=0.125, workspace=ws), o, kappa, A, want)
    assert ops.workspace_status(ws) == 2 + 8
    wd.copy_(w)
    ws = paged.evict_workspace(3, hkv, 10, "cuda")
    new = paged.kv_evict(kd, vd, wd, td, nd, 10, workspace=ws)
    assert new.tolist() == [10, 10, 0]
    assert ops.workspace_status(ws) == 2 + 8
    used = set(table[0, [0, 2]].tolist()) | set(table[1].tolist())
    others = [p for p in range(k.shape[0]) if p not in used]
    assert torch.equal(words(kd)[others], words(k)[others]) and torch.equal(wd.cpu()[others], w[others])


@pytest.mark.gpu
def test_infinities_and_nan():
    """A NaN or an infinity in a visible row shows where the definition shows it, and in no other sequence or head."""
    from lara_b200 import paged

    hq, hkv, d, page = 4, 2, 64, 16
    k, v, table, n = make_cache([300, 300, 300, 300], hkv, d, page, seed=6, shared=2)
    q = torch.randn((4, hq, d), generator=torch.Generator().manual_seed(1)).bfloat16()
    at = lambda b, t: (int(table[b, t // page]), 0, t % page)  # noqa: E731
    v[at(0, 299)][5] = math.nan
    v[at(1, 130)][7] = math.inf
    k[at(2, 77)][3] = math.nan
    w = torch.zeros(k.shape[:3])
    for scored in (True, False):
        qd, kd, vd, wd, td, nd = dev(q, k, v, w, table, n)
        if scored:
            got = paged.gqa_decode_scored(qd, kd, vd, wd, td, nd)  # shared pages: their weights are not looked at
        else:
            got = paged.gqa_decode_shared(qd, kd, vd, td, nd, 2)
        bad = ~torch.isfinite(got.float().cpu())
        want = torch.zeros_like(bad)
        want[0, :2, 5] = want[1, :2, 7] = True
        want[2, :2] = True
        assert torch.equal(bad, want)
    v[at(3, 3)] = math.nan  # in the shared part: in every sequence's first kv head
    got = paged.gqa_decode_shared(qd, k.cuda(), v.cuda(), td, nd, 2).float().cpu()
    assert torch.isnan(got[:, :2]).all() and torch.isfinite(got[[0, 1, 2, 3], 2:]).all()


@pytest.mark.gpu
def test_graphs_streams_and_views():
    """Calls captured in two graphs with a workspace each, replayed in turn; another stream; 16-bit views."""
    from lara_b200 import paged

    hq, hkv, d, page = 16, 2, 128, 64
    k, v, table, n = make_cache([700, 513, 90], hkv, d, page, seed=12, shared=1)
    q = torch.randn((2, 3, hq, d), generator=torch.Generator().manual_seed(2)).bfloat16()
    w = torch.rand(k.shape[:3], generator=torch.Generator().manual_seed(3))
    qd, kd, vd, wd, td, nd = dev(q, k, v, w, table, n)
    k2, v2, t2, n2 = dev(*make_cache([700, 513, 90], hkv, d, page, seed=12))
    w2 = torch.rand(k2.shape[:3], device="cuda")
    runs = []
    for i in range(2):
        ws = (paged.shared_workspace(3, hq, hkv, d, "cuda"), paged.scored_workspace(3, hq, k2, t2.shape[1]),
              paged.evict_workspace(3, hkv, 300, "cuda"))
        keep = [x.clone() for x in (k2, v2, w2)]
        out = [torch.empty_like(qd[i]) for _ in range(2)]
        w_out, src, new = torch.empty_like(w2), torch.empty((3, hkv, 300), dtype=torch.int32, device="cuda"), n2.clone()
        w_out.copy_(w2)

        def call(i=i, ws=ws, keep=keep, out=out, w_out=w_out, src=src, new=new):
            paged.gqa_decode_shared(qd[i], kd, vd, td, nd, 1, workspace=ws[0], out=out[0])
            paged.gqa_decode_scored(qd[i], keep[0], keep[1], keep[2], t2, n2, weights_out=w_out, workspace=ws[1],
                                    out=out[1])
            paged.kv_evict(keep[0], keep[1], w_out, t2, n2, 300, first=1, last=9, new_lens=new, sources=src,
                           workspace=ws[2])

        runs.append((call, keep, out, w_out, src, new))
    want = []
    for call, keep, out, w_out, src, new in runs:
        call()
        torch.cuda.synchronize()
        want.append([x.clone() for x in (*keep, *out, w_out, src, new)])
    graphs = []
    for call, keep, *_ in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)

    def reset():
        for _, keep, out, w_out, src, new in runs:
            for x, y in zip(keep, (k2, v2, w2)):
                x.copy_(y)
            w_out.copy_(w2)
            for x in (*out, src, new):
                x.zero_()

    def check():
        torch.cuda.synchronize()
        for (_, keep, out, w_out, src, new), ref in zip(runs, want):
            for x, y in zip((*keep, *out, w_out, src, new), ref):
                assert torch.equal(words(x), words(y))

    for order in ((0, 1), (1, 0)):
        reset()
        for i in order:
            graphs[i].replay()
        check()
    reset()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for s, g in zip(streams, graphs):  # at the same time
        with torch.cuda.stream(s):
            g.replay()
    check()
    reset()
    torch.cuda.synchronize()
    for s, (call, *_) in zip(streams, runs):
        with torch.cuda.stream(s):
            call()
    check()
    view = paged.gqa_decode_shared(qd[0].view(torch.int16), kd.view(torch.int16), vd.view(torch.int16), td, nd, 1)
    assert torch.equal(view.cpu(), words(runs[0][2][0]))


@pytest.mark.gpu
def test_rows_past_32_bit_offsets():
    """Pages whose elements lie past 2^32 in the pool."""
    from lara_b200 import paged

    hq, hkv, d, page = 8, 4, 128, 256
    num = (1 << 32) // (hkv * page * d) + 40  # 2^32 elements and some pages
    lens = [900, 300, 513]
    k, v, table, n = make_cache(lens, hkv, d, page, seed=21)
    used = k.shape[0]
    big = [torch.empty((num, hkv, page, d), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    w = torch.rand(k.shape[:3], generator=torch.Generator().manual_seed(3))
    w_big = torch.zeros((num, hkv, page), device="cuda")
    for x, y in zip((*big, w_big), (k, v, w)):
        x[num - used:] = y.cuda()
    there = torch.where(table >= 0, table + (num - used), table)
    q = torch.randn((3, hq, d), generator=torch.Generator().manual_seed(5)).bfloat16()
    o, kappa, A, ps = decode64(q, k, v, table, n, page, d ** -0.5)
    td, nd, qd = dev(there, n, q)
    check_out(paged.gqa_decode_shared(qd, *big, td, nd, 0), o, kappa, A, n)
    check_out(paged.gqa_decode_scored(qd, *big, w_big, td, nd), o, kappa, A, n)
    check_weights(w_big[num - used:], w, ps, A, table, n, page, d)
    w = w_big[num - used:].cpu()
    want = evict64(k, v, w, table, n, page, 200, 4, 30)
    paged.kv_evict(*big, w_big, td, nd, 200, first=4, last=30)
    for x, y in zip((*big, w_big), want):
        assert torch.equal(words(x[num - used:]), words(y))
    k, v, table, n = make_cache([900, 800], hkv, d, page, seed=22, shared=3)
    used = k.shape[0]
    for x, y in zip(big, (k, v)):
        x[num - used:] = y.cuda()
    there = torch.where(table >= 0, table + (num - used), table)
    o, kappa, A, _ = decode64(q[:2], k, v, table, n, page, d ** -0.5)
    check_out(paged.gqa_decode_shared(qd[:2].contiguous(), *big, there.cuda(), n.cuda(), 3), o, kappa, A, n)


@pytest.mark.gpu
def test_scored_decode_names_more_pages_than_there_are():
    """Sequences that share pages: the output is right, weights past the room are left and flagged."""
    from lara_b200 import ops, paged

    hq, hkv, d, page = 4, 1, 64, 16
    k, v, table, n = make_cache([320], hkv, d, page, seed=30)
    table, n = table.repeat(40, 1), n.repeat(40)
    q = torch.randn((40, hq, d), generator=torch.Generator().manual_seed(1)).bfloat16()
    o, kappa, A, _ = decode64(q, k, v, table, n, page, 0.125)
    qd, kd, vd, td, nd = dev(q, k, v, table, n)
    ws = paged.scored_workspace(40, hq, kd, table.shape[1])
    wd = torch.zeros(k.shape[:3], device="cuda")
    check_out(paged.gqa_decode_scored(qd, kd, vd, wd, td, nd, scale=0.125, workspace=ws), o, kappa, A, n)
    assert ops.workspace_status(ws) == 32


@pytest.mark.gpu
def test_many_sequences():
    """More sequences than cached lengths and than threads that count them, most of them short or empty."""
    from lara_b200 import paged

    hq, hkv, d, page = 4, 2, 64, 16
    g = torch.Generator().manual_seed(17)
    lens = torch.randint(0, 40, (2500,), generator=g).tolist()
    lens[1700] = 2000
    lens[:300] = [0] * 300
    k, v, table, n = make_cache(lens, hkv, d, page, seed=3)
    q = torch.randn((len(lens), hq, d), generator=g).bfloat16()
    w = torch.rand(k.shape[:3], generator=g)
    o, kappa, A, ps = decode64(q, k, v, table, n, page, 0.125)
    qd, kd, vd, wd, td, nd = dev(q, k, v, w, table, n)
    check_out(paged.gqa_decode_shared(qd, kd, vd, td, nd, 0, scale=0.125), o, kappa, A, n)
    check_out(paged.gqa_decode_scored(qd, kd, vd, wd, td, nd, scale=0.125), o, kappa, A, n)
    check_weights(wd, w, ps, A, table, n, page, d)
    w = wd.cpu()
    want = evict64(k, v, w, table, n, page, 20, 2, 3)
    paged.kv_evict(kd, vd, wd, td, nd, 20, first=2, last=3)
    for x, y in zip((kd, vd, wd), want):
        assert torch.equal(words(x), words(y))
    k, v, table, n = make_cache([64 + x for x in lens], hkv, d, page, seed=5, shared=4)
    o, kappa, A, _ = decode64(q, k, v, table, n, page, 0.125)
    qd, kd, vd, td, nd = dev(q, k, v, table, n)
    check_out(paged.gqa_decode_shared(qd, kd, vd, td, nd, 4, scale=0.125), o, kappa, A, n)


# ------------------------------------------------------------------ refusals
BAD_CFG, DEST, RESULT, UNSUPPORTED = 0x01, 0x11, 0x12, 0x22
P = 1 << 20  # an address that is aligned and never used: every call here is refused on the host


def c_call(name, **change):
    """A valid call's arguments with some replaced; the status code."""
    from lara_b200._native import lib

    pool = dict(n_kv_heads=2, head_dim=64, page_size=16, pages_per_seq=4, num_pages=9)
    if name == "evict":
        a = dict(k=P, v=P, w=P, w_out=P, table=P, lens=P, new_lens=2 * P, sources=0, batch=3, **pool, keep=8, first=1,
                 last=2, ws=P, nbytes=1 << 40, stream=0)
        fn = lib.lara_kv_evict
    elif name == "scored":
        a = dict(q=P, k=P, v=P, w=P, w_out=P, table=P, lens=P, o=P, batch=3, n_q_heads=8, **pool, scale=0.5, ws=P,
                 nbytes=1 << 40, stream=0)
        fn = lib.lara_gqa_decode_scored
    else:
        a = dict(q=P, k=P, v=P, table=P, lens=P, o=P, batch=3, n_q_heads=8, **pool, shared=1, scale=0.5, ws=P,
                 nbytes=1 << 40, stream=0)
        fn = lib.lara_gqa_decode_shared
    assert set(change) <= set(a)
    a.update(change)
    return fn(*a.values())


EVERY = [(dict(head_dim=96), UNSUPPORTED), (dict(page_size=8), BAD_CFG), (dict(page_size=48), BAD_CFG),
         (dict(batch=-1), BAD_CFG), (dict(batch=65536), BAD_CFG), (dict(n_kv_heads=0), BAD_CFG),
         (dict(num_pages=0), BAD_CFG), (dict(pages_per_seq=0), BAD_CFG), (dict(pages_per_seq=1 << 26), BAD_CFG),
         (dict(batch=65535, n_kv_heads=8, pages_per_seq=1 << 25, n_q_heads=8), BAD_CFG),
         (dict(k=0), DEST), (dict(v=0), DEST), (dict(table=0), DEST), (dict(lens=0), DEST), (dict(ws=0), DEST),
         (dict(k=P + 8), DEST), (dict(v=P + 2), DEST), (dict(table=P + 2), DEST), (dict(lens=P + 1), DEST),
         (dict(ws=P + 16), DEST), (dict(nbytes=256), RESULT), (dict(nbytes=0), RESULT)]
DECODE = [(dict(n_q_heads=0), BAD_CFG), (dict(n_q_heads=7), BAD_CFG), (dict(n_q_heads=34), UNSUPPORTED),
          (dict(scale=0.0), BAD_CFG), (dict(scale=-1.0), BAD_CFG), (dict(scale=math.nan), BAD_CFG),
          (dict(scale=math.inf), BAD_CFG), (dict(q=0), DEST), (dict(o=0), DEST), (dict(q=P + 8), DEST),
          (dict(o=P + 4), DEST)]
WEIGHTS = [(dict(w=0), DEST), (dict(w_out=0), DEST), (dict(w=P + 4), DEST), (dict(w_out=P + 8), DEST),
           (dict(w_out=P + 64), DEST)]


@pytest.mark.parametrize("name", ["shared", "scored", "evict"])
def test_refused_on_the_host(name):
    own = {"shared": DECODE + [(dict(shared=-1), BAD_CFG), (dict(shared=5), BAD_CFG)], "scored": DECODE + WEIGHTS,
           "evict": WEIGHTS + [(dict(keep=0), BAD_CFG), (dict(first=-1), BAD_CFG), (dict(last=-1), BAD_CFG),
                               (dict(first=6, last=3), BAD_CFG), (dict(first=9), BAD_CFG),
                               (dict(first=0x7fffffff, last=0x7fffffff), BAD_CFG), (dict(new_lens=P), DEST),
                               (dict(new_lens=P + 8), DEST), (dict(sources=P + 2), DEST),
                               (dict(pages_per_seq=(1 << 20) + 1), UNSUPPORTED),
                               (dict(num_pages=1 << 30, n_kv_heads=4), BAD_CFG)]}[name]
    for change, code in EVERY + own:
        if name == "evict":
            change = {x: y for x, y in change.items() if x != "n_q_heads"}
        assert c_call(name, **change) == code, change
    assert c_call(name, batch=0, k=0, v=0, table=0, ws=0) == 0  # nothing to do


def test_workspaces_serve_smaller_calls():
    from lara_b200._native import lib

    for d in (64, 128):
        for hkv in (1, 2, 8):
            for group in (1, 5, 8, 16):
                sizes = [lib.lara_decode_shared_workspace_bytes(b, hkv * group, hkv, d) for b in range(1, 300, 7)]
                assert sizes == sorted(sizes) and sizes[0] > 0
                assert lib.lara_decode_shared_workspace_bytes(64, hkv, hkv, d) <= \
                    lib.lara_decode_shared_workspace_bytes(64, hkv * group, hkv, d)
                sizes = [lib.lara_decode_scored_workspace_bytes(b, hkv * group, hkv, d, 16, 100, 900)
                         for b in range(1, 300, 7)]
                assert sizes == sorted(sizes) and sizes[0] > 0
    assert lib.lara_kv_evict_workspace_bytes(2, 8, 100) < lib.lara_kv_evict_workspace_bytes(3, 8, 101)
    for bad in ((0, 8, 2, 64), (3, 0, 2, 64), (3, 8, 0, 64)):
        assert lib.lara_decode_shared_workspace_bytes(*bad) == 0
    assert lib.lara_kv_evict_workspace_bytes(3, 2, 0) == 0


def test_refused_by_the_binding():
    """What the Python binding refuses before any address is used (CPU tensors stand for the wrong device)."""
    from lara_b200 import paged

    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    q, w = torch.zeros((1, 8, 64), dtype=torch.bfloat16), torch.zeros((4, 2, 16))
    table, n, ws = torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(4096)
    with pytest.raises(TypeError, match="k_pages must hold bf16"):
        paged.gqa_decode_shared(q, k.float(), k, table, n, 1, workspace=ws)
    with pytest.raises(ValueError, match="k_pages must be on the CUDA device"):
        paged.gqa_decode_shared(q, k, k, table, n, 1, workspace=ws)
    with pytest.raises(ValueError, match="num_pages, Hkv, page_size, D"):
        paged.gqa_decode_scored(q, k[0], k, w, table, n, workspace=ws)
    with pytest.raises(ValueError, match="k_pages must be on the CUDA device"):
        paged.kv_evict(k, k, w, table, n, 3, workspace=ws)
    with pytest.raises(TypeError, match="must be a tensor"):
        paged.kv_evict(None, k, w, table, n, 3, workspace=ws)


@pytest.mark.gpu
def test_refused_tensors():
    from lara_b200 import paged
    from lara_b200._native import LaraConfigError
    from lara_b200.kvquant import QuantKVCache

    k, v, table, n = dev(*make_cache([40, 20], 2, 64, 16, seed=1))
    q = torch.zeros((2, 8, 64), dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(k.shape[:3], device="cuda")
    ws = paged.shared_workspace(2, 8, 2, 64, "cuda")
    ok = dict(q=q, k=k, v=v, table=table, n=n, shared=0)

    def shared(**change):
        a = {**ok, **change}
        return paged.gqa_decode_shared(a["q"], a["k"], a["v"], a["table"], a["n"], a["shared"],
                                       scale=a.get("scale"), workspace=a.get("ws", ws), out=a.get("out"))

    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    for error, change in [(ValueError, dict(q=q[:, :, :32])), (ValueError, dict(q=q[0])),
                          (TypeError, dict(q=q.float())), (ValueError, dict(q=q.cpu())), (ValueError, dict(q=turned)),
                          (ValueError, dict(v=v[:1])), (ValueError, dict(k=k[:, :, ::2], v=v[:, :, ::2])),
                          (ValueError, dict(table=table.long())), (ValueError, dict(table=table[:1])),
                          (ValueError, dict(table=table.t().contiguous().t())), (ValueError, dict(n=n.long())),
                          (ValueError, dict(n=n[:1])), (ValueError, dict(shared=-1)), (ValueError, dict(shared=99)),
                          (TypeError, dict(shared=1.5)), (ValueError, dict(scale=0.0)), (TypeError, dict(scale="x")),
                          (ValueError, dict(out=q[:1])), (ValueError, dict(ws=ws[:256])),
                          (ValueError, dict(ws=ws.cpu())),
                          (ValueError, dict(out=q[:, :1].expand(2, 8, 64)))]:
        with pytest.raises(error):
            shared(**change)
    with pytest.raises(ValueError):
        paged.gqa_decode_scored(q, k, v, w[:1], table, n)
    with pytest.raises(TypeError):
        paged.gqa_decode_scored(q, k, v, w.half(), table, n)
    for change in (dict(keep=0), dict(keep=3, first=2, last=2), dict(keep=3, new_lens=n), dict(keep=3, first=-1),
                   dict(keep=4, sources=torch.zeros((2, 2, 3), dtype=torch.int32, device="cuda"))):
        with pytest.raises((ValueError, LaraConfigError)):
            paged.kv_evict(k, v, w, table, n, change.pop("keep"), **change)
    assert shared(q=q[:0], table=table[:0], n=n[:0]).shape == (0, 8, 64)
    cache = paged.PagedKVCache(8, 16, 2, 64, 3, 64, "cuda")
    cache.new_sequence()
    with pytest.raises(ValueError, match="scored=True"):
        cache.decode_scored(q[:1])
    with pytest.raises(ValueError, match="scored=True"):
        cache.evict(3)
    with pytest.raises(ValueError, match="bf16"):
        quant = QuantKVCache(8, 16, 2, 64, 3, 64, "cuda")
        quant.new_sequence()
        quant.decode_shared(q[:1])
    cache = paged.PagedKVCache(12, 16, 2, 64, 3, 64, "cuda", scored=True)
    rows = torch.zeros((1, 2, 40, 64), dtype=torch.bfloat16, device="cuda")
    cache.new_sequence(), cache.new_sequence()
    cache.append(rows, rows, [0])
    cache.share_prefix(0, 1, 40)
    for call in (lambda: cache.decode_scored(q), lambda: cache.evict(8), lambda: cache.evict(8, [0])):
        with pytest.raises(ValueError, match="in common"):
            call()
    cache.free_sequence(1)
    with pytest.raises(ValueError, match="twice"):
        cache.evict(8, [0, 0])
    cache.decode_scored(q[:1])
    assert cache.weights.sum() > 7  # eight heads' weights
    cache.reserve([0], 20)
    free = cache.free_pages
    cache.evict(60)
    assert cache.free_pages == free and cache.seq_len(0) == 40  # nothing cut, nothing freed
    cache.evict(30)
    cache.new_sequence()
    with pytest.raises(ValueError, match="cut"):
        cache.share_prefix(0, 1, 16)
    cache.free_sequence(1)
    cache.free_sequence(0)
    cache.new_sequence()
    cache.append(rows, rows, [0])
    cache.new_sequence()
    assert cache.share_prefix(0, 1, 16) == 16
    assert not cache.weights[cache.block_table[0, :3].long()].any()  # pages start anew
