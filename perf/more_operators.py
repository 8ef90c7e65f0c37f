"""Cases of the operators that serve many or long sequences from a paged bf16 cache.

* ``shared``: one new token per sequence, of a batch whose sequences begin with the same cached pages;
* ``scored``: one new token per sequence, and every cached slot's attention weight of this step added to what it
  has gathered so far (the sum over the query heads of its kv head);
* ``evict``: every sequence and kv head is cut down to its first slots, its last ones and the heaviest of the
  rest; kept rows from behind move into the freed slots.

``run`` makes one pass: in elementary torch operations where ``own`` is false, through ``lara_b200.paged`` where
it is true.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # a few users of one assistant prompt (latency)
        dict(name="shared_few", op="shared", batch=4, hq=32, hkv=8, d=128, page=64, prefix=1024, n=48, ragged=True,
             short=False),
        # a serving batch behind a long common document
        dict(name="shared_batch", op="shared", batch=64, hq=32, hkv=8, d=128, page=256, prefix=8192, n=512,
             ragged=True, short=False),
        # an odd batch, five heads to a kv head, small pages, sequences among it that end within the prefix
        dict(name="shared_odd", op="shared", batch=37, hq=10, hkv=2, d=64, page=16, prefix=2000, n=333, ragged=True,
             short=True),
        # many samples of one long context
        dict(name="shared_samples", op="shared", batch=256, hq=64, hkv=8, d=128, page=256, prefix=16384, n=1024,
             ragged=True, short=False),
        # one conversation (latency)
        dict(name="scored_one", op="scored", batch=1, hq=32, hkv=8, d=128, page=64, n=500, ragged=False),
        # a serving batch: 64 sequences of 4096 tokens, 32 query heads on 8 kv heads
        dict(name="scored_batch", op="scored", batch=64, hq=32, hkv=8, d=128, page=256, n=4096, ragged=False),
        # a ragged batch, an empty sequence among it, head_dim 64, seven heads to a kv head
        dict(name="scored_ragged", op="scored", batch=33, hq=28, hkv=4, d=64, page=32, n=9000, ragged=True),
        # one long context, groups of 8 heads
        dict(name="scored_long", op="scored", batch=1, hq=64, hkv=8, d=128, page=256, n=524288, ragged=False),
        # a step of a batch at its budget: one slot of each kv head goes (latency)
        dict(name="evict_step", op="evict", batch=16, hkv=8, d=128, page=64, n=2049, keep=2048, first=4, last=256,
             ragged=False),
        # prompts cut to a quarter after prefill
        dict(name="evict_prompts", op="evict", batch=32, hkv=8, d=128, page=256, n=8192, keep=2048, first=4, last=512,
             ragged=False),
        # an odd budget, ragged lengths (some below it), small pages, head_dim 64
        dict(name="evict_odd", op="evict", batch=33, hkv=2, d=64, page=16, n=3001, keep=777, first=1, last=33,
             ragged=True),
        # one long context cut to an eighth
        dict(name="evict_long", op="evict", batch=1, hkv=8, d=128, page=256, n=524288, keep=65536, first=16, last=1024,
             ragged=False),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["shared", "scored", "evict"])
    d = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128, 256])
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8, 16])
    ragged = rng.random() < 0.6
    if op == "shared":
        batch = _between(rng, 1, 256)
        n = _between(rng, 1, min(4096, 262144 // batch))
        prefix = page * _between(rng, 1, max(1, min(32768, (1 << 28) // (batch * hkv * group)) // page))
        return dict(op=op, batch=batch, hq=hkv * group, hkv=hkv, d=d, page=page, prefix=prefix, n=n, ragged=ragged,
                    short=rng.random() < 0.3)
    if op == "scored":
        tokens = min(524288, (1 << 25) // (hkv * group))  # of the whole batch
        n = _between(rng, 1, min(262144, tokens))
        return dict(op=op, batch=_between(rng, 1, min(256, tokens // n)), hq=hkv * group, hkv=hkv, d=d, page=page,
                    n=n, ragged=ragged)
    n = _between(rng, 2, 262144)
    keep = _between(rng, 1, n)
    first = min(keep, rng.choice([0, 1, 4, 16]))
    return dict(op=op, batch=_between(rng, 1, min(256, 262144 // n)), hkv=hkv, d=d, page=page, n=n, keep=keep,
                first=first, last=rng.choice([0, (keep - first) // 8, (keep - first) // 2]), ragged=ragged)


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _lens(g, case):
    """Sequence lengths (own tokens): all n, or ragged, spread evenly up to n, one empty among three or more."""
    B, n = case["batch"], case["n"]
    if not case["ragged"]:
        return [n] * B
    lens = [max(1, n * (i + 1) // B) for i in range(B)]
    if B > 2:
        lens[B // 2] = 0
    return [lens[i] for i in torch.randperm(B, generator=g, device=DEV).tolist()]


def _pool(g, pages, case):
    """K and V pages of unit normal rows; four channels of K ten times as large, as keys have them."""
    shape = (pages, case["hkv"], case["page"], case["d"])
    out = []
    for _ in range(2):
        x = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
        step = max(1, (1 << 25) // (shape[1] * shape[2] * shape[3]))
        for p in range(0, pages, step):
            y = torch.randn((min(step, pages - p), *shape[1:]), generator=g, device=DEV)
            if not out:
                y[..., 3::shape[3] // 4] *= 10.0
            x[p:p + step] = y
        out.append(x)
    return out


def _weights(g, pages, case):
    """What slots have gathered: a heavy tail, a twentieth of them nothing at all (ties)."""
    shape = (pages, case["hkv"], case["page"])
    w = torch.exp(2.0 * torch.randn(shape, generator=g, device=DEV)) / case["n"]
    return torch.where(torch.rand(shape, generator=g, device=DEV) < 0.05, 0.0, w)


def _inputs(case, seed):
    g = _gen(seed)
    ps = case["page"]
    own_lens = _lens(g, case)
    shared = case["prefix"] // ps if case["op"] == "shared" else 0
    lens = [shared * ps + n for n in own_lens] if shared else own_lens
    if shared and case["short"]:
        for b in range(1, len(lens), 5):  # some end within the prefix, or have nothing
            lens[b] = lens[b] * 7919 % (shared * ps + 1)
    per_seq = max(1, -(-max(lens) // ps))
    used = [max(0, -(-n // ps) - shared) for n in lens]
    pages = max(1, shared + sum(used))
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), per_seq), -1, dtype=torch.int32, device=DEV)
    table[:, :shared] = perm[:shared]
    at = shared
    for b, u in enumerate(used):
        table[b, shared:shared + u] = perm[at:at + u]
        at += u
    k, v = _pool(g, pages, case)
    s = dict(k=k, v=v, table=table, lens=_i32(lens), lens_host=lens)
    if case["op"] != "evict":
        q = torch.randn((case["batch"], case["hq"], case["d"]), generator=g, device=DEV)
        s["q"] = q.to(torch.bfloat16)
    if case["op"] != "shared":
        s["w"] = _weights(g, pages, case)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    op = case["op"]
    if op != "shared":
        s["w_out"] = s["w"].clone()
    if op == "evict":
        s["new_lens"] = torch.empty_like(s["lens"])
        s["sources"] = torch.empty((case["batch"], case["hkv"], case["keep"]), dtype=torch.int32, device=DEV)
    if own:
        from lara_b200 import paged

        if op == "shared":
            s["workspace"] = paged.shared_workspace(case["batch"], case["hq"], case["hkv"], case["d"], DEV)
        elif op == "scored":
            s["workspace"] = paged.scored_workspace(case["batch"], case["hq"], s["k"], s["table"].shape[1])
        else:
            s["workspace"] = paged.evict_workspace(case["batch"], case["hkv"], case["keep"], DEV)
        if op != "evict":
            s["out"] = torch.empty_like(s["q"])
    return s


# --------------------------------------------------------------------------- one pass
def run(state):
    return _PASS[state["case"]["op"]][bool(own)](state)


def _rows(s, x, b, lo, hi):
    """fp32 [hkv, hi - lo, d] of tokens lo .. hi - 1 of sequence b; lo on a page's border."""
    ps = s["case"]["page"]
    pages = s["table"][b, lo // ps:-(-hi // ps)].long()
    return x[pages].float().transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :hi - lo]


def _softmax(x):
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _shared_plain(s):
    case = s["case"]
    B, hq, hkv, d, P = case["batch"], case["hq"], case["hkv"], case["d"], case["prefix"]
    G = hq // hkv
    kp, vp = _rows(s, s["k"], 0, 0, P), _rows(s, s["v"], 0, 0, P)
    q = s["q"].float().view(B, hkv, G, d) * (1.0 / math.sqrt(d))
    o = torch.zeros((B, hkv, G, d), dtype=torch.float32, device=DEV)
    step = max(1, (1 << 28) // (hq * P))  # sequences at a time
    for b0 in range(0, B, step):
        qs = q[b0:b0 + step]
        sp = torch.matmul(qs.transpose(0, 1).reshape(hkv, -1, d), kp.transpose(1, 2))
        sp = sp.view(hkv, -1, G, P)
        for i in range(qs.shape[0]):
            n = s["lens_host"][b0 + i]
            if n == 0:
                continue
            x = sp[:, i, :, :min(n, P)]
            if n > P:
                x = torch.cat([x, torch.matmul(qs[i], _rows(s, s["k"], b0 + i, P, n).transpose(1, 2))], -1)
            x = _softmax(x)
            y = torch.matmul(x[..., :P], vp[:, :min(n, P)])
            if n > P:
                y = y + torch.matmul(x[..., P:], _rows(s, s["v"], b0 + i, P, n))
            o[b0 + i] = y
    return o.view(B, hq, d).to(torch.bfloat16)


def _shared_own(s):
    from lara_b200 import paged

    return paged.gqa_decode_shared(s["q"], s["k"], s["v"], s["table"], s["lens"],
                                   s["case"]["prefix"] // s["case"]["page"], workspace=s["workspace"], out=s["out"])


def _scored_plain(s):
    case = s["case"]
    hkv, d, ps = case["hkv"], case["d"], case["page"]
    o = torch.zeros(s["q"].shape, dtype=torch.float32, device=DEV)
    for b, n in enumerate(s["lens_host"]):
        if n == 0:
            continue
        q = s["q"][b].float().view(hkv, -1, d) * (1.0 / math.sqrt(d))
        p = _softmax(torch.matmul(q, _rows(s, s["k"], b, 0, n).transpose(1, 2)))
        o[b] = torch.matmul(p, _rows(s, s["v"], b, 0, n)).view(-1, d)
        t = torch.arange(n, device=DEV)
        page, row = s["table"][b].long()[t // ps], t % ps
        s["w_out"][page, :, row] = s["w"][page, :, row] + p.sum(1).t()
    return o.to(torch.bfloat16), s["w_out"]


def _scored_own(s):
    from lara_b200 import paged

    o = paged.gqa_decode_scored(s["q"], s["k"], s["v"], s["w"], s["table"], s["lens"], weights_out=s["w_out"],
                                workspace=s["workspace"], out=s["out"])
    return o, s["w_out"]


def _evict_plain(s):
    case = s["case"]
    keep, first, last, ps = case["keep"], case["first"], case["last"], case["page"]
    k, v, w, w_out, src = s["k"], s["v"], s["w"], s["w_out"], s["sources"]
    at = torch.arange(keep, device=DEV)
    for b, n in enumerate(s["lens_host"]):
        t = torch.arange(n, device=DEV)
        page, row = s["table"][b].long()[t // ps], t % ps
        if n <= keep:
            src[b] = torch.where(at < n, at, -1)
            w_out[page, :, row] = w[page, :, row]
            continue
        have = w[page, :, row].t()
        x = torch.where((t < first) | (t >= n - last), math.inf, have)
        kept = torch.zeros(have.shape, dtype=torch.bool, device=DEV)
        kept.scatter_(1, torch.sort(x, descending=True, stable=True).indices[:, :keep], True)
        h, holes = torch.nonzero(~kept[:, :keep], as_tuple=True)  # as many of a head as of the next line
        movers = torch.nonzero(kept[:, keep:], as_tuple=True)[1] + keep
        k[page[holes], h, row[holes]] = k[page[movers], h, row[movers]]
        v[page[holes], h, row[holes]] = v[page[movers], h, row[movers]]
        src[b] = at
        src[b, h, holes] = movers.int()
        w_out[page[:keep], :, row[:keep]] = have.gather(1, src[b].long()).t()
        w_out[page[keep:], :, row[keep:]] = 0.0
    s["new_lens"].copy_(torch.clamp(s["lens"], max=keep))
    return k, v, w_out, s["new_lens"], src


def _evict_own(s):
    from lara_b200 import paged

    case = s["case"]
    paged.kv_evict(s["k"], s["v"], s["w"], s["table"], s["lens"], case["keep"], first=case["first"],
                   last=case["last"], weights_out=s["w_out"], new_lens=s["new_lens"], sources=s["sources"],
                   workspace=s["workspace"])
    return s["k"], s["v"], s["w_out"], s["new_lens"], s["sources"]


_PASS = {
    "shared": (_shared_plain, _shared_own),
    "scored": (_scored_plain, _scored_own),
    "evict": (_evict_plain, _evict_own),
}


# --------------------------------------------------------------------------- work
def work(case):
    B, hkv, d, n = case["batch"], case["hkv"], case["d"], case["n"]
    tokens = B * n // (2 if case["ragged"] and B > 1 else 1)  # ragged: about half of the longest
    if case["op"] == "evict":
        keep, first, last = case["keep"], case["first"], case["last"]
        moved = 0.0
        if n > keep:
            rest = (keep - first - last) / (n - first - last)  # of the unprotected slots, those that stay
            behind = n - keep
            moved = min(last, behind) + rest * max(0, behind - last)
        moved *= hkv * tokens / n
        return dict(bytes=moved * 8 * d + 8 * tokens * hkv + 4 * B * hkv * keep, flops=tokens * hkv)
    hq = case["hq"]
    prefix = case.get("prefix", 0)
    moved = 4 * d * hkv * (prefix + tokens) + 4 * B * hq * d
    if case["op"] == "scored":
        moved += 8 * tokens * hkv
    return dict(bytes=moved, flops=4 * d * hq * (B * prefix + tokens))


# --------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](case, s)


def _whole(x, pages, h, n):
    """fp64 [n, d] of one sequence's first n tokens of kv head h."""
    return torch.cat([x[p, h] for p in pages.split(4096)]).reshape(-1, x.shape[-1])[:n].double()


def _attention(case, s, given=None):
    """o in fp64; `given` gets the weights of each (sequence, kv head), summed over the heads."""
    d, ps, hkv = case["d"], case["page"], case["hkv"]
    G = case["hq"] // hkv
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for h in range(hkv):
        last = None
        for b, n in enumerate(s["lens_host"]):
            if n == 0:
                continue
            pages = s["table"][b, :-(-n // ps)].long()
            front = case.get("prefix", 0)
            if front and n >= front:  # the common rows are turned into fp64 once
                if last is None:
                    last = [_whole(x, pages[:front // ps], h, front) for x in (s["k"], s["v"])]
                rest = pages[front // ps:]
                k, v = ([x, _whole(y, rest, h, n - front)] if n > front else [x]
                        for x, y in zip(last, (s["k"], s["v"])))
            else:
                k, v = ([_whole(x, pages, h, n)] for x in (s["k"], s["v"]))
            q = s["q"][b, h * G:(h + 1) * G].double() / math.sqrt(d)
            logits = torch.cat([q @ x.T for x in k], -1)
            w = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
            parts = w.split([x.shape[0] for x in v], -1)
            o[b, h * G:(h + 1) * G] = sum(a @ x for a, x in zip(parts, v))
            if given is not None:
                given(b, h, n, w.sum(0))
    return o


def _exact_shared(case, s):
    return _attention(case, s)


def _exact_scored(case, s):
    w = s["w"].double()
    ps = case["page"]

    def add(b, h, n, x):
        pages = s["table"][b, :-(-n // ps)].long()
        x = torch.nn.functional.pad(x, (0, pages.numel() * ps - n)).view(-1, ps)
        w[:, h].index_add_(0, pages, x)

    return _attention(case, s, add), w


def _exact_evict(case, s):
    keep, first, last, ps = case["keep"], case["first"], case["last"], case["page"]
    k, v, w = s["k"], s["v"], s["w"].double()
    src = torch.full((case["batch"], case["hkv"], keep), -1, dtype=torch.int64, device=DEV)
    for b, n in enumerate(s["lens_host"]):
        src[b, :, :min(n, keep)] = torch.arange(min(n, keep), device=DEV)
        if n <= keep:
            continue
        pages = s["table"][b, :-(-n // ps)].long()
        for h in range(case["hkv"]):
            have = w[pages, h].reshape(-1)[:n]
            free = keep - first - last
            middle = have[first:n - last]
            stays = torch.ones(n, dtype=torch.bool, device=DEV)
            if free == 0:
                stays[first:n - last] = False
            else:
                # every weight above the border, and of those at it the lowest slots
                border = torch.sort(middle).values[middle.numel() - free]
                above, equal = middle > border, middle == border
                room = free - int(above.sum())
                stays[first:n - last] = above | (equal & (torch.cumsum(equal, 0) <= room))
            empty = torch.nonzero(~stays[:keep]).flatten()
            come = torch.nonzero(stays[keep:]).flatten() + keep
            src[b, h, empty] = come
            to, of = (pages[empty // ps], h, empty % ps), (pages[come // ps], h, come % ps)
            for x in (k, v):
                x[to] = x[of]
            new = torch.zeros_like(have)
            new[:keep] = have[src[b, h]]
            all_ = torch.arange(n, device=DEV)
            w[pages[all_ // ps], h, all_ % ps] = new
    return k, v, w, torch.clamp(s["lens"].long(), max=keep), src


_EXACT = {"shared": _exact_shared, "scored": _exact_scored, "evict": _exact_evict}
