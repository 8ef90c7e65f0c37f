"""Cases of the 8-bit KV cache operators and of the q/k norm with rotation.

Four operators of a serving step with a quantised cache:

* ``norm_rope``: RMS norm of every query and key head and the position rotation, in one pass;
* ``append``: new K/V rows are quantised as they are written into a paged pool (one row, the
  ``head_dim`` values of one token and kv head, has 8-bit codes and one fp32 scale), then the
  rows just written are read back, since 8-bit contents are compared as the values they stand for;
* ``read``: cached rows are turned back into bf16, contiguous per sequence, for the bf16 kernels;
* ``decode``: one new token per sequence attends its cached tokens.

``run`` makes one pass: in elementary torch operations where ``own`` is false, through
``lara_b200`` where it is true.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
MAX_POS = 131072
EPS = 1e-5
TINY = 2.0 ** -100


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a small batch: q/k heads of single tokens at scattered positions (latency)
        dict(name="norm_rope_step", op="norm_rope", tokens=8, hq=32, hkv=8, d=128, rot=128, interleaved=True,
             packed=True, prompt=False),
        # a prompt of odd length, head_dim 64, half-rotated heads, pairs half a rotation apart
        dict(name="norm_rope_prompt_odd", op="norm_rope", tokens=1999, hq=8, hkv=2, d=64, rot=32, interleaved=False,
             packed=False, prompt=True),
        # several prompts of a prefill pass at once, q and k read out of the projection's packed output
        dict(name="norm_rope_prefill", op="norm_rope", tokens=16384, hq=64, hkv=8, d=128, rot=128, interleaved=False,
             packed=True, prompt=True),
        # one decode step of a serving batch: a row per sequence and kv head (latency)
        dict(name="append_step", op="append", batch=64, n=1, hkv=8, d=128, page=64, fmt="int8", ragged=False,
             token_major=True, cached=4096),
        # a few prompts of different lengths padded to the longest, small pages
        dict(name="append_ragged", op="append", batch=5, n=517, hkv=2, d=64, page=16, fmt="fp8_e4m3", ragged=True,
             token_major=False, cached=1000),
        # a prefill chunk of 2048 tokens for each of 8 sequences, 8192 cached
        dict(name="append_chunk", op="append", batch=8, n=2048, hkv=8, d=128, page=256, fmt="int8", ragged=False,
             token_major=False, cached=8192),
        # a short prefix read back, ragged
        dict(name="read_prefix", op="read", batch=3, n=700, hkv=8, d=128, page=64, fmt="fp8_e4m3", ragged=True),
        # the cached part of a chunked prefill: 8192 tokens of each of 8 sequences
        dict(name="read_long", op="read", batch=8, n=8192, hkv=8, d=128, page=256, fmt="int8", ragged=False),
        # one short conversation (latency)
        dict(name="decode_one", op="decode", batch=1, n=300, hq=32, hkv=8, d=128, page=64, fmt="int8", ragged=False),
        # a serving batch: 64 sequences of 4096 tokens, 32 query heads on 8 kv heads
        dict(name="decode_batch", op="decode", batch=64, n=4096, hq=32, hkv=8, d=128, page=256, fmt="int8",
             ragged=False),
        # a ragged batch, an empty sequence among them, groups of 8 heads
        dict(name="decode_ragged", op="decode", batch=32, n=32768, hq=64, hkv=8, d=128, page=64, fmt="fp8_e4m3",
             ragged=True),
        # one context of a million tokens
        dict(name="decode_long", op="decode", batch=1, n=1048576, hq=32, hkv=8, d=128, page=256, fmt="int8",
             ragged=False),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "read", "decode", "decode"])
    d = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128, 256])
    fmt = rng.choice(["int8", "fp8_e4m3"])
    if op == "norm_rope":
        hq, hkv = rng.choice([(32, 8), (64, 8), (8, 2), (16, 16), (40, 8)])
        return dict(op=op, tokens=_between(rng, 1, 16384), hq=hq, hkv=hkv, d=d, rot=rng.choice([d, d // 2]),
                    interleaved=rng.random() < 0.5, packed=rng.random() < 0.5, prompt=rng.random() < 0.5)
    if op == "append":
        n = rng.choice([1, _between(rng, 1, 4096)])
        return dict(op=op, batch=_between(rng, 1, min(256, 16384 // n)), n=n, hkv=rng.choice([1, 2, 8]), d=d,
                    page=page, fmt=fmt, ragged=rng.random() < 0.5, token_major=rng.random() < 0.5,
                    cached=rng.randrange(0, 8192))
    if op == "read":
        n = _between(rng, 1, 16384)
        return dict(op=op, batch=_between(rng, 1, min(64, 65536 // n)), n=n, hkv=rng.choice([1, 2, 8]), d=d,
                    page=page, fmt=fmt, ragged=rng.random() < 0.5)
    n = _between(rng, 1, 262144)
    hkv, group = rng.choice([1, 2, 8]), rng.choice([1, 2, 4, 5, 8, 16])
    return dict(op=op, batch=_between(rng, 1, max(1, min(256, 524288 // n))), n=n, hq=hkv * group, hkv=hkv, d=d,
                page=page, fmt=fmt, ragged=rng.random() < 0.5)


# --------------------------------------------------------------------------- quantised rows, in torch
def _quantise(x, fmt):
    """bf16 rows [..., d] -> (codes in the pool's type, fp32 scales [...])."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(x).all(-1, keepdim=True)
    if fmt == "int8":
        a = amax.clamp_min(TINY)
        scale = a / 127.0
        codes = torch.where(finite, torch.round(x * 127.0 / a), 0.0).to(torch.int8)
    else:
        m, e = torch.frexp(amax)
        e = torch.where(m <= 0.875, e - 9, e - 8).clamp_min(-100)
        scale = torch.ldexp(torch.ones_like(amax), e)
        codes = torch.where(finite, x / scale, 0.0).to(torch.float8_e4m3fn)
    return codes, torch.where(finite, scale, math.nan).squeeze(-1)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _rows(g, shape, d):
    """bf16 K or V rows: unit normal, four channels of the head ten times as large (as keys have them)."""
    x = torch.randn((*shape, d), generator=g, device=DEV)
    x[..., 3:d:d // 4] *= 10.0
    return x.to(torch.bfloat16)


def _pool(g, pages, case):
    """A pool whose every row holds a quantised row, made in pieces of a few hundred MB."""
    hkv, ps, d, fmt = case["hkv"], case["page"], case["d"], case["fmt"]
    dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    codes = torch.empty((pages, hkv, ps, d), dtype=dt, device=DEV)
    scales = torch.empty((pages, hkv, ps), dtype=torch.float32, device=DEV)
    step = max(1, (1 << 25) // (hkv * ps * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        c, s = _quantise(_rows(g, (n, hkv, ps), d), fmt)
        codes[p:p + n].view(torch.int8).copy_(c.view(torch.int8))
        scales[p:p + n] = s
    return codes, scales


def _tables(g, lens, capacity, page):
    """A block table of pages in random order, -1 past each sequence's last page; the number of pages."""
    per_seq = (capacity + page - 1) // page
    used = [(n + page - 1) // page for n in lens]
    perm = torch.randperm(max(1, sum(used)), generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), per_seq), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        at += u
    return table, max(1, sum(used))


def _lens(g, case):
    """Sequence lengths: all n, or ragged (the first n long, one empty among three or more)."""
    B, n = case["batch"], case["n"]
    if not case["ragged"]:
        return [n] * B
    lens = torch.randint(1, n + 1, (B,), generator=g, device=DEV).tolist()
    lens[0] = n
    if B > 2:
        lens[B // 2] = 0
    return lens


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# --------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "norm_rope":
        T, hq, hkv, d, rot = case["tokens"], case["hq"], case["hkv"], case["d"], case["rot"]
        x = torch.randn((T, hq + 2 * hkv, d), generator=g, device=DEV)
        x *= 0.5 + 2.0 * torch.rand((1, hq + 2 * hkv, 1), generator=g, device=DEV)
        x = x.to(torch.bfloat16)
        q, k = x[:, :hq], x[:, hq:hq + hkv]
        if not case["packed"]:
            q, k = q.contiguous(), k.contiguous()
        if case["prompt"]:
            start = int(torch.randint(0, MAX_POS - T, (1,), generator=g, device=DEV))
            pos = torch.arange(start, start + T, device=DEV)
        else:
            pos = torch.randint(0, MAX_POS, (T,), generator=g, device=DEV)
        i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
        ang = torch.arange(MAX_POS, dtype=torch.float64, device=DEV)[:, None] * (10000.0 ** (-2.0 * i / rot))
        w = 1.0 + 0.2 * torch.randn((2, d), generator=g, device=DEV)
        return dict(q=q, k=k, positions=pos.to(torch.int32), qw=w[0].to(torch.bfloat16), kw=w[1].to(torch.bfloat16),
                    cos_sin=torch.cat([ang.cos(), ang.sin()], -1).float())
    if op == "append":
        B, n, hkv, d = case["batch"], case["n"], case["hkv"], case["d"]
        starts = torch.randint(0, case["cached"] + 1, (B,), generator=g, device=DEV).tolist()
        counts = _lens(g, case)
        shape = (B, n, hkv) if case["token_major"] else (B, hkv, n)
        k, v = _rows(g, shape, d), _rows(g, shape, d)
        if case["token_major"]:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        table, pages = _tables(g, [s + c for s, c in zip(starts, counts)], case["cached"] + n, case["page"])
        kc, ks = _pool(g, pages, dict(case, page=case["page"]))
        vc, vs = kc.clone(), ks.clone()
        return dict(k=k, v=v, starts=_i32(starts), counts=_i32(counts), table=table, kc=kc, vc=vc, ks=ks, vs=vs)
    lens = _lens(g, case)
    table, pages = _tables(g, lens, max(lens), case["page"])
    kc, ks = _pool(g, pages, case)
    vc, vs = _pool(g, pages, case)
    out = dict(table=table, lens=_i32(lens), lens_host=lens, kc=kc, vc=vc, ks=ks, vs=vs)
    if op == "decode":
        out["q"] = torch.randn((case["batch"], case["hq"], case["d"]), generator=g, device=DEV).to(torch.bfloat16)
    return out


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        from lara_b200 import kvquant

        if case["op"] == "norm_rope":
            s["out"] = tuple(torch.empty(t.shape, dtype=t.dtype, device=DEV) for t in (s["q"], s["k"]))
            return s
        s["pool"] = kvquant.QuantPool(s["kc"], s["vc"], s["ks"], s["vs"])
        if case["op"] == "decode":
            s["workspace"] = kvquant.decode_workspace(case["batch"], case["hq"], case["hkv"], case["d"], DEV)
            s["out"] = torch.empty_like(s["q"])
        else:
            shape = (case["batch"], case["hkv"], case["n"], case["d"])
            s["out"] = tuple(torch.empty(shape, dtype=torch.bfloat16, device=DEV) for _ in range(2))
            s["new_lens"] = torch.empty((case["batch"],), dtype=torch.int32, device=DEV)
    return s


# --------------------------------------------------------------------------- one pass
def run(state):
    return _PASS[state["case"]["op"]][bool(own)](state)


def _norm_rope_plain(s):
    d, rot, inter = s["case"]["d"], s["case"]["rot"], s["case"]["interleaved"]
    cs = s["cos_sin"][s["positions"].long()]
    cos, sin = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
    outs = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        x = x.float()
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        if inter:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = y[..., :rot // 2], y[..., rot // 2:rot]
            r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        outs.append(torch.cat([r, y[..., rot:]], -1).to(torch.bfloat16))
    return tuple(outs)


def _norm_rope_own(s):
    from lara_b200 import ops

    return ops.qk_norm_rope(s["q"], s["k"], positions=s["positions"], cos_sin=s["cos_sin"], q_weight=s["qw"],
                            k_weight=s["kw"], eps=EPS, interleaved=s["case"]["interleaved"], out=s["out"])


def _read_plain(s, lens, starts):
    """bf16 k, v [B, hkv, n, d] of tokens starts .. starts + n - 1, zeros at and past lens."""
    n, ps = s["case"]["n"], s["case"]["page"]
    pos = starts.long()[:, None] + torch.arange(n, device=DEV)
    valid = pos < lens.long()[:, None]
    pos = torch.where(valid, pos, 0)
    page = torch.where(valid, s["table"].long().gather(1, pos // ps), 0)
    outs = []
    for codes, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        x = codes.view(torch.int8)[page, :, pos % ps].view(codes.dtype).float() * scales[page, :, pos % ps, None]
        x = torch.where(valid[:, :, None, None], x, 0.0)
        outs.append(x.to(torch.bfloat16).transpose(1, 2).contiguous())
    return tuple(outs)


def _append_plain(s):
    case = s["case"]
    n, ps = case["n"], case["page"]
    i = torch.arange(n, device=DEV)
    b, i = torch.nonzero(i < s["counts"].long()[:, None], as_tuple=True)
    pos = s["starts"].long()[b] + i
    page, row = s["table"].long()[b, pos // ps], pos % ps
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        c, sc = _quantise(x[b, :, i], case["fmt"])
        codes.view(torch.int8)[page, :, row] = c.view(torch.int8)
        scales[page, :, row] = sc
    lens = s["starts"] + s["counts"]
    return (*_read_plain(s, lens, s["starts"]), lens)


def _append_own(s):
    from lara_b200 import kvquant

    kvquant.kvq_append(s["pool"], s["table"], s["starts"], s["k"], s["v"], counts=s["counts"],
                       new_lens=s["new_lens"])
    k, v = kvquant.kvq_read(s["pool"], s["table"], s["new_lens"], s["case"]["n"], starts=s["starts"], out=s["out"])
    return k, v, s["new_lens"]


def _read_only_plain(s):
    return _read_plain(s, s["lens"], torch.zeros_like(s["lens"]))


def _read_own(s):
    from lara_b200 import kvquant

    return kvquant.kvq_read(s["pool"], s["table"], s["lens"], s["case"]["n"], out=s["out"])


def _decode_plain(s):
    case = s["case"]
    hkv, d, ps = case["hkv"], case["d"], case["page"]
    group = case["hq"] // hkv
    o = torch.zeros(s["q"].shape, dtype=torch.float32, device=DEV)
    for b, n in enumerate(s["lens_host"]):
        if n == 0:
            continue
        pages = s["table"][b, :(n + ps - 1) // ps].long()

        def rows(codes, scales):
            x = codes.view(torch.int8)[pages].view(codes.dtype).float() * scales[pages][..., None]
            return x.transpose(0, 1).reshape(hkv, -1, d)[:, :n]

        q = s["q"][b].float().view(hkv, group, d)
        p = torch.matmul(q, rows(s["kc"], s["ks"]).transpose(1, 2)) * (1.0 / math.sqrt(d))
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o[b] = torch.matmul(p, rows(s["vc"], s["vs"])).view(-1, d)
    return o.to(torch.bfloat16)


def _decode_own(s):
    from lara_b200 import kvquant

    return kvquant.gqa_decode_kvq(s["q"], s["pool"], s["table"], s["lens"], workspace=s["workspace"], out=s["out"])


_PASS = {
    "norm_rope": (_norm_rope_plain, _norm_rope_own),
    "append": (_append_plain, _append_own),
    "read": (_read_only_plain, _read_own),
    "decode": (_decode_plain, _decode_own),
}


# --------------------------------------------------------------------------- work
def work(case):
    op, d, hkv = case["op"], case["d"], case["hkv"]
    if op == "norm_rope":
        n = case["tokens"] * (case["hq"] + hkv) * d
        return dict(bytes=4 * n + case["tokens"] * (4 * case["rot"] + 4) + 4 * d, flops=9 * n)
    if op in ("append", "read"):
        # with ragged lengths, about half of the rows are there; the outputs are written whole
        rows = 2 * case["batch"] * case["n"] * hkv
        have = rows // 2 if case["ragged"] else rows
        moved = have * (d + 4) + rows * d * 2  # the cache's rows read, the bf16 rows written
        if op == "append":
            moved += have * d * 2 + have * (d + 4)  # the bf16 rows read, the cache's rows written
        return dict(bytes=moved, flops=(3 if op == "append" else 1) * have * d)
    tokens = case["batch"] * case["n"] // (2 if case["ragged"] and case["batch"] > 1 else 1)
    return dict(bytes=2 * tokens * hkv * (d + 4) + 4 * case["batch"] * case["hq"] * d,
                flops=4 * tokens * case["hq"] * d)


# --------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](case, s)


def _exact_norm_rope(case, s):
    d, rot = case["d"], case["rot"]
    half = rot // 2
    cs = s["cos_sin"].double()[s["positions"].long()]
    first = torch.arange(half, device=DEV) * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)
    outs = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = torch.empty(x.shape, dtype=torch.float64, device=DEV)
        for t in range(0, x.shape[0], 4096):
            z = x[t:t + 4096].double()
            z = z * (z.square().sum(-1, keepdim=True) / d + EPS).rsqrt() * w.double()
            turn = torch.complex(cs[t:t + 4096, None, :half], cs[t:t + 4096, None, half:])
            z2 = torch.complex(z[..., first], z[..., second]) * turn
            z[..., first], z[..., second] = z2.real, z2.imag
            y[t:t + 4096] = z
        outs.append(y)
    return tuple(outs)


def _exact_values(x, fmt):
    """What the quantised form of rows x stands for."""
    x = x.double()
    top = x.abs().max(-1, keepdim=True).values
    if fmt == "int8":
        top = torch.maximum(top, torch.full_like(top, TINY))
        return torch.round(127.0 * x / top) * (top / 127.0)
    s = torch.exp2(torch.ceil(torch.log2(torch.maximum(top, torch.full_like(top, TINY)) / 448.0)).clamp_min(-100.0))
    y = x / s
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(y / step) * step * s


def _exact_append(case, s):
    n = case["n"]
    there = (torch.arange(n, device=DEV) < s["counts"][:, None])[:, None, :, None]
    k, v = (torch.where(there, _exact_values(x, case["fmt"]), 0.0).contiguous() for x in (s["k"], s["v"]))
    return k, v, s["starts"] + s["counts"]


def _exact_row_values(codes, scales, pages, n):
    """fp64 [hkv, n, d] of one sequence's first n tokens."""
    parts = [codes[p].double() * scales[p].double()[..., None] for p in pages]
    return torch.cat(parts, 1)[:, :n]


def _exact_read(case, s):
    shape = (case["batch"], case["hkv"], case["n"], case["d"])
    outs = []
    for codes, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        y = torch.zeros(shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(s["lens_host"]):
            if n:
                pages = s["table"][b, :-(-n // case["page"])].tolist()
                y[b, :, :n] = _exact_row_values(codes, scales, pages, n)
        outs.append(y)
    return tuple(outs)


def _exact_decode(case, s):
    d, ps, hkv = case["d"], case["page"], case["hkv"]
    group = case["hq"] // hkv
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lens_host"]):
        if n == 0:
            continue
        pages = s["table"][b, :-(-n // ps)].long()
        for h in range(hkv):
            def flat(codes, scales):
                x = codes.view(torch.int8)[pages, h].view(codes.dtype).double()
                return (x * scales[pages, h].double()[..., None]).reshape(-1, d)[:n]

            q = s["q"][b, h * group:(h + 1) * group].double()
            logits = q @ flat(s["kc"], s["ks"]).T / math.sqrt(d)
            weights = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
            o[b, h * group:(h + 1) * group] = weights @ flat(s["vc"], s["vs"])
    return o


_EXACT = {"norm_rope": _exact_norm_rope, "append": _exact_append, "read": _exact_read, "decode": _exact_decode}
