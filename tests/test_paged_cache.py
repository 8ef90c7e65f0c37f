"""What ``PagedKVCache`` keeps of its sequences beside the kernels' work: pages, prefixes, files, status.

On the CPU the kernels' workspaces are plain memory, and no kernel runs.
"""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_paged_serving import check_out, check_weights, decode64  # noqa: E402


@pytest.fixture
def cpu_cache(monkeypatch):
    from lara_b200 import paged

    monkeypatch.setattr(paged, "new_workspace",
                        lambda nbytes, device: torch.zeros(max(int(nbytes), 256), dtype=torch.uint8, device=device))

    def make(num_pages, page_size, max_seqs, max_seq_len, **kw):
        return paged.PagedKVCache(num_pages, page_size, 2, 64, max_seqs, max_seq_len, "cpu", **kw)

    return make


def hold(cache, slot, n):
    """n more tokens without their rows."""
    cache.reserve([slot], n)
    cache._lens[slot] += n
    cache._sync_rows([slot])


def consistent(cache):
    assert torch.equal(cache.block_table.cpu(), torch.from_numpy(cache._table))
    assert torch.equal(cache.lens.cpu(), torch.from_numpy(cache._lens))
    taken = cache._table[cache._table >= 0]
    assert np.array_equal(np.bincount(taken, minlength=cache.num_pages), cache._refs)
    assert sorted(cache._free) == np.flatnonzero(cache._refs == 0).tolist()


# ------------------------------------------------------------------ pages
def test_reserve_that_is_refused_takes_no_pages(cpu_cache):
    cache = cpu_cache(5, 16, 3, 64, scored=True)
    cache.weights += 3.0  # what earlier sequences gathered
    a, b = cache.new_sequence(), cache.new_sequence()
    hold(cache, a, 32), hold(cache, b, 32)
    cache.weights += 3.0
    before = cache._table.copy(), cache.weights.clone()
    with pytest.raises(MemoryError):
        cache.reserve([a, b], 1)  # one page is left for two
    with pytest.raises(ValueError, match="capacity"):
        hold(cache, b, 16), cache.reserve([a, b], 17)
    cache.free_sequence(b)
    assert np.array_equal(cache._table[a], before[0][a])
    consistent(cache)
    b = cache.new_sequence()
    cache.reserve([a, b, a], 1)
    consistent(cache)
    new = [int(cache._table[a, 2]), int(cache._table[b, 0])]
    assert not cache.weights[new].any()
    assert torch.equal(cache.weights[cache._table[a, :2]], before[1][cache._table[a, :2]])
    assert cache.free_pages == 1


@pytest.mark.gpu
def test_append_again_after_the_pool_was_exhausted():
    from lara_b200.paged import PagedKVCache

    hq, hkv, d, page = 8, 2, 64, 16
    g = torch.Generator().manual_seed(4)
    rows = lambda b, n: torch.randn((b, hkv, n, d), generator=g).bfloat16().cuda()  # noqa: E731
    query = lambda b: torch.randn((b, hq, d), generator=g).bfloat16().cuda()  # noqa: E731
    cache = PagedKVCache(6, page, hkv, d, 3, 64, "cuda", scored=True)
    for _ in range(3):
        cache.new_sequence()
    cache.append(rows(3, 32), rows(3, 32))
    cache.decode_scored(query(3))  # every page has weights
    cache.free_sequence(2)
    cache.append(rows(1, 16), rows(1, 16), [0])  # one page is left
    with pytest.raises(MemoryError):
        cache.append(rows(2, 1), rows(2, 1), [0, 1])
    assert cache.free_pages == 1
    cache.evict(16, [0])
    cache.append(rows(2, 1), rows(2, 1), [0, 1])
    consistent(cache)
    lens, table = cache.lens[:2].cpu(), cache.block_table.cpu()
    assert lens.tolist() == [17, 33]
    before = cache.weights.cpu()
    assert not before[table[0, 1], :, 0].any() and not before[table[1, 2]].any()
    q = query(2)
    o, kappa, A, ps = decode64(q.cpu(), cache.k_pages.cpu(), cache.v_pages.cpu(), table, lens, page, d ** -0.5)
    check_out(cache.decode_shared(q), o, kappa, A, lens)
    check_out(cache.decode_scored(q), o, kappa, A, lens)
    check_weights(cache.weights, before, ps, A, table, lens, page, d)
    assert cache.status() == 0


# ------------------------------------------------------------------ status
@pytest.mark.gpu
@pytest.mark.parametrize("call", ["decode", "decode_shared", "decode_scored", "evict", "quant"])
def test_status_outlasts_the_workspace(call):
    """A bad page that a small call met is reported also when a larger call has come since."""
    from lara_b200.kvquant import QuantKVCache
    from lara_b200.paged import PagedKVCache

    hkv, d, page = 1, 64, 16
    if call == "quant":
        cache = QuantKVCache(400, page, hkv, d, 40, 1 << 16, "cuda")
    else:
        cache = PagedKVCache(400, page, hkv, d, 40, 1 << 16, "cuda", scored=True)
    for _ in range(40):
        cache.new_sequence()
    rows = torch.zeros((40, hkv, 20, d), dtype=torch.bfloat16, device="cuda")
    cache.append(rows, rows)

    def go(slots, heads):
        if call == "evict":
            cache.evict(18 + heads // 8, slots)
        else:
            q = torch.zeros((len(slots), heads, d), dtype=torch.bfloat16, device="cuda")
            getattr(cache, "decode" if call == "quant" else call)(q, slots)

    good = cache.block_table.clone()
    cache.block_table[0, 0] = 1 << 20
    go([0], 1)
    small = cache._ws if call in ("decode", "quant") else cache._serving_ws[call.removeprefix("decode_")]
    cache.block_table.copy_(good)
    more = torch.zeros((1, hkv, 4000, d), dtype=torch.bfloat16, device="cuda")
    cache.append(more, more, [39])
    go(list(range(40)), 8)
    assert small is not (cache._ws if call in ("decode", "quant") else cache._serving_ws[call.removeprefix("decode_")])
    assert cache.status() == 8 and cache.status() == 0


# ------------------------------------------------------------------ files
def test_files_say_which_sequences_are_cut(tmp_path):
    from lara_b200 import kvfile

    g = np.random.default_rng(1)
    k, v = (g.integers(0, 1 << 16, (3, 2, 5, 64), dtype=np.uint16) for _ in "kv")
    lens = np.array([5, 0, 3], np.int32)
    whole, cut = tmp_path / "whole.npz", tmp_path / "cut.npz"
    kvfile.save(whole, k, v, lens, np.zeros(3, bool))
    with np.load(whole) as z:
        assert "cut" not in z  # as before
    kvfile.save(cut, k, v, lens, np.array([False, False, True]))
    for x, y in zip(kvfile.load(whole), (k, v, lens)):
        assert np.array_equal(x, y)
    for path, want in ((whole, [0, 0, 0]), (cut, [0, 0, 1])):
        for x, y in zip(kvfile.load_any(path), (k, v, lens, np.array(want, bool))):
            assert np.array_equal(x, y)
    with pytest.raises(ValueError, match=r"\[2\] have been cut"):
        kvfile.load(cut)
    with np.load(cut) as z:
        held = dict(z)
    for change in (dict(cut=np.array([True, False, True])), dict(cut=None)):
        np.savez(cut, **{x: y for x, y in {**held, **change}.items() if y is not None})
        with pytest.raises(ValueError, match="checksum"):
            kvfile.load_any(cut)
    with pytest.raises(ValueError, match="cut"):
        kvfile.save(cut, k, v, lens, np.ones(2, bool))


@pytest.mark.gpu
def test_a_cut_sequence_from_a_file_is_nobodys_prefix(tmp_path):
    from lara_b200.attn_driver import AttentionAccelerator
    from lara_b200.paged import PagedKVCache

    cache = PagedKVCache(24, 16, 2, 64, 6, 64, "cuda", scored=True)
    g = torch.Generator().manual_seed(2)
    for n in (40, 33):
        s = cache.new_sequence()
        rows = torch.randn((1, 2, n, 64), generator=g).bfloat16().cuda()
        cache.append(rows, rows, [s])
    cache.decode_scored(torch.randn((2, 4, 64), generator=g).bfloat16().cuda())
    cache.evict(32, [0])
    cache.save(tmp_path / "kv")
    a, b = cache.load(tmp_path / "kv")
    for x, y in zip((*cache.gather(a), *cache.gather(b)), (*cache.gather(0), *cache.gather(1))):
        assert torch.equal(x, y)
    c = cache.new_sequence()
    with pytest.raises(ValueError, match="cut"):
        cache.share_prefix(a, c, 16)
    assert cache.share_prefix(b, c, 33) == 32
    with AttentionAccelerator() as acc:
        acc.configure_heads(4, 2, 64, max_seq_len=64, batch=2)
        with pytest.raises(ValueError, match="cut"):
            acc.restore_kv(tmp_path / "kv")
    cache.free_sequence(a)
    assert cache.new_sequence() == a  # whole again
    rows = torch.zeros((1, 2, 20, 64), dtype=torch.bfloat16, device="cuda")
    cache.append(rows, rows, [a])
    assert cache.share_prefix(a, cache.new_sequence(), 16) == 16


# ------------------------------------------------------------------ common prefixes
def most_spared(rows, lens, page):
    """The definition of ``shared_pages``, prefix by prefix."""
    best, pages = 0, 0
    for n in range(1, max(lens) // page + 1):
        holders = [r[:n].tolist() for r, m in zip(rows, lens) if m // page >= n]
        if all(x == holders[0] for x in holders) and n * (len(holders) - 1) > best:
            best, pages = n * (len(holders) - 1), n
    return pages


def test_shared_pages_leaves_short_sequences_aside(cpu_cache):
    cache = cpu_cache(400, 16, 40, 640)
    doc = cache.new_sequence()
    hold(cache, doc, 330)
    group = [doc]
    for n in range(5):
        s = cache.new_sequence()
        assert cache.share_prefix(doc, s, 330) == 320
        if n:
            hold(cache, s, 17 * n)
        group.append(s)
    assert cache.shared_pages() == cache.shared_pages(group) == 20
    empty, short, other = cache.new_sequence(), cache.new_sequence(), cache.new_sequence()
    hold(cache, short, 100)  # pages of its own, fewer than the prefix has
    assert cache.shared_pages([empty] + group) == cache.shared_pages(group + [empty, short]) == 20
    inside = cache.new_sequence()
    assert cache.share_prefix(doc, inside, 200) == 192
    assert cache.shared_pages([inside] + group) == 20
    hold(cache, other, 321)  # as long, and other pages
    assert cache.shared_pages(group + [other]) == 0
    assert cache.shared_pages([empty, short]) == cache.shared_pages([empty, cache.new_sequence()]) == 0
    assert cache.shared_pages([doc]) == 21 and cache.shared_pages([empty]) == 0
    assert cache.shared_pages([short, short]) == 6  # whole pages


def test_shared_pages_of_any_slots(cpu_cache):
    rng = np.random.default_rng(7)
    for _ in range(60):
        cache = cpu_cache(600, 16, 12, 320)
        slots = []
        for i in range(12):
            s = cache.new_sequence()
            if slots and rng.random() < 0.7:
                src = int(rng.choice(slots))
                cache.share_prefix(src, s, int(rng.integers(0, cache.seq_len(src) + 1)))
            hold(cache, s, int(rng.integers(0, 321 - cache.seq_len(s)) * rng.random()))
            slots.append(s)
        for _ in range(8):
            pick = rng.choice(slots, rng.integers(2, 13), replace=bool(rng.random() < 0.3))
            want = most_spared(cache._table[pick], [cache.seq_len(s) for s in pick], 16)
            assert cache.shared_pages(pick) == want


@pytest.mark.gpu
def test_decode_shared_beside_sequences_that_end_within_the_prefix():
    """An empty slot, a short sequence, and one that shares less read for themselves what the others read together."""
    from lara_b200 import paged

    hq, hkv, d, page = 8, 2, 64, 16
    g = torch.Generator().manual_seed(6)
    rows = lambda n: torch.randn((1, hkv, n, d), generator=g).bfloat16().cuda()  # noqa: E731
    cache = paged.PagedKVCache(64, page, hkv, d, 8, 400, "cuda")
    doc = cache.new_sequence()
    x = rows(200)
    cache.append(x, x, [doc])
    for n in (0, 5, 40):
        s = cache.new_sequence()
        assert cache.share_prefix(doc, s, 200) == 192
        if n:
            x = rows(n)
            cache.append(x, x, [s])
    cache.new_sequence()
    short = cache.new_sequence()
    x = rows(70)
    cache.append(x, x, [short])
    assert cache.share_prefix(doc, cache.new_sequence(), 100) == 96
    assert cache.shared_pages() == 12
    q = torch.randn((7, hq, d), generator=g).bfloat16()
    lens = torch.tensor([200, 192, 197, 232, 0, 70, 96])
    o, kappa, A, _ = decode64(q, cache.k_pages.cpu(), cache.v_pages.cpu(), cache.block_table.cpu(), lens, page, d ** -0.5)
    check_out(cache.decode_shared(q.cuda()), o, kappa, A, lens)
    assert cache.status() == 0


# ------------------------------------------------------------------ refusals
def test_8_bit_cache_names_what_it_lacks():
    from lara_b200.kvquant import QuantKVCache

    cache = QuantKVCache.__new__(QuantKVCache)  # before any memory is asked for
    cache.weights = None
    q = torch.zeros((1, 8, 64), dtype=torch.bfloat16)
    for call in (lambda: cache.decode_scored(q), lambda: cache.decode_shared(q), lambda: cache.evict(8)):
        with pytest.raises(ValueError, match="bf16 rows"):
            call()


def test_evict_refuses_outputs_over_what_it_reads():
    from test_paged_serving import DEST, P, c_call

    # 3 sequences, 4 pages each, 2 kv heads, 8 slots kept: 12 bytes of lengths, 48 of table, 192 of sources
    far = dict(table=3 * P, lens=4 * P, new_lens=5 * P, sources=6 * P)
    for change in (dict(new_lens=4 * P + 8), dict(new_lens=4 * P - 8), dict(new_lens=3 * P + 44), dict(new_lens=3 * P - 8),
                   dict(sources=3 * P + 44), dict(sources=3 * P - 188), dict(sources=4 * P + 8), dict(sources=4 * P - 188),
                   dict(sources=5 * P + 8), dict(sources=5 * P - 188)):
        assert c_call("evict", **{**far, **change}) == DEST, change
    # next to each other they are accepted, and refused for the workspace alone
    for change in (dict(new_lens=4 * P + 12), dict(new_lens=3 * P + 48), dict(sources=3 * P - 192), dict(sources=5 * P + 12),
                   dict(sources=4 * P - 192), dict(new_lens=0, sources=0)):
        assert c_call("evict", **{**far, **change}, nbytes=0) == 0x12, change


def test_evict_names_its_bound_of_units():
    from lara_b200._native import lib
    from test_paged_serving import BAD_CFG, c_call

    few = dict(page_size=16, pages_per_seq=1, num_pages=1, nbytes=0)
    assert c_call("evict", **few, batch=1 << 15, n_kv_heads=1 << 12) == BAD_CFG
    assert b"below 2^27" in lib.lara_last_error_string()
    assert c_call("evict", **few, batch=(1 << 15) - 1, n_kv_heads=1 << 12) == 0x12  # the workspace alone
