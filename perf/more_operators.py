"""What the operators of a decoding loop are judged on, next to the cache's own: many continuations
of a prompt, with drafted tokens, a step at a time without the host between. One operator a case:

* ``share``: ``morpho_cache_attention`` over sequences that have a long prefix in common (the full
  pages that forks share). ``groups`` prompts of ``shortest`` to ``prefix`` tokens with ``members``
  sequences each, and ``alone`` sequences that share with nobody; every sequence has ``rest_least`` to
  ``rest_most`` tokens of its own behind, then ``new`` new ones (fewer where ``ragged``); ``heads``,
  ``cube`` (codes per head), ``head_dim`` (value columns per head), ``page`` (tokens a page); ``mask``:
  ``causal``, or ``tree`` (the new tokens are drafts that see their ancestors);
* ``verify``: ``morpho_verify_drafts``: ``batch`` sequences of ``new`` tokens (the last decided one and
  drafts) against the target's logits over ``vocab`` tokens; ``shape``: ``chain`` or ``tree``; ``drawn``:
  the drafts were drawn from the drafter's distributions (else they were its best guesses);
  ``temperature`` (0: the best token decides);
* ``plan``: ``morpho_cache_plan``: the pages of a step's new tokens and where each goes, and then the
  pages back that the kept ones do not need: ``batch`` sequences of ``shortest`` to ``longest`` tokens
  and up to ``new`` new ones, of which up to ``keep`` stay; ``spare``: pages that are free, for each 100
  that the step asks for.
"""

from __future__ import annotations

import math
import random

import torch

DEVICE = "cuda"

# set by the harness: the framework's kernels instead of the plain forms
own = False

_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_NONE = -torch.finfo(torch.float32).max


def _share(name, groups, members, alone, new, shortest, prefix, rest_least, rest_most, heads, cube, head_dim, *,
           page=64, mask="causal", ragged=False, scale=1.0):
    c = {"op": "share", "groups": groups, "members": members, "alone": alone, "new": new, "shortest": shortest,
         "prefix": prefix, "rest_least": rest_least, "rest_most": rest_most, "heads": heads, "cube": cube,
         "head_dim": head_dim, "page": page, "mask": mask, "ragged": ragged, "scale": scale}
    return {**c, "name": name} if name else c


def _verify(name, batch, new, vocab, dtype, *, shape="chain", drawn=True, temperature=1.0, ragged=False):
    c = {"op": "verify", "batch": batch, "new": new, "vocab": vocab, "dtype": dtype, "shape": shape, "drawn": drawn,
         "temperature": temperature, "ragged": ragged}
    return {**c, "name": name} if name else c


def _plan(name, batch, shortest, longest, new, keep, *, page=64, spare=100, ragged=False):
    c = {"op": "plan", "batch": batch, "shortest": shortest, "longest": longest, "new": new, "keep": keep, "page": page,
         "spare": spare, "ragged": ragged}
    return {**c, "name": name} if name else c


def listed():
    return [
        # the next token of a small beam through the smallest module of the tests: launches and their latency
        _share("share_beam", 1, 4, 0, 1, 256, 256, 1, 20, 8, 16, 32),
        # 64 answers to one long prompt through the headline module
        _share("share_samples", 1, 64, 0, 1, 8192, 8192, 1, 500, 16, 16, 64),
        # several users' prompts with as many answers each, and users who share with nobody
        _share("share_prompts", 4, 12, 16, 1, 700, 4096, 5, 1000, 16, 32, 64, scale=0.5),
        # a tree of drafts for each of 16 answers of the widest module
        _share("share_tree", 1, 16, 0, 48, 4096, 4096, 20, 600, 32, 64, 64, mask="tree", ragged=True, scale=0.125),
        # 32 questions about one very long document
        _share("share_document", 1, 32, 0, 1, 65536, 65536, 10, 1000, 16, 32, 64, scale=0.5),
        # four drafts of one user: launches, and the chain of decisions
        _verify("verify_one", 1, 5, 32000, "float16"),
        # five drafts of each of 64 users, of a large vocabulary
        _verify("verify_batch", 64, 6, 128000, "bfloat16", temperature=0.8),
        # a tree of the drafter's best guesses for each of 16 users, an odd vocabulary
        _verify("verify_tree", 16, 48, 50001, "float16", shape="tree", drawn=False, ragged=True),
        # trees of drafts that were drawn, several of one place: each that is turned down leaves another remainder
        _verify("verify_siblings", 8, 24, 32001, "float32", shape="tree", temperature=0.7),
        # no randomness: the best token decides
        _verify("verify_best", 32, 8, 65536, "bfloat16", temperature=0.0),
        # a step of drafts of 64 users in the middle of their conversations
        _plan("plan_drafts", 64, 1, 8191, 12, 12),
        # prompts of many users at once, and none of them kept
        _plan("plan_prompts", 512, 0, 0, 2000, 0, ragged=True, spare=90),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["share", "share", "share", "verify", "verify", "plan"])
    if op == "plan":
        batch = _log_int(rng, 1, 2000)
        new = max(1, min(_log_int(rng, 1, 2000), 1000000 // batch))
        longest = _log_int(rng, 1, 8000)
        return _plan(None, batch, rng.randint(0, longest), longest, new, rng.randint(0, new),
                     page=rng.choice([32, 64, 64, 128, 256]), spare=rng.choice([0, 60, 100, 100, 150]),
                     ragged=rng.random() < 0.6)
    if op == "verify":
        dtype, shape = rng.choice(["float16", "bfloat16", "float32"]), rng.choice(["chain", "tree"])
        drawn = rng.random() < 0.6
        vocab = _log_int(rng, 100, 140000)
        new = rng.randint(1, 12) if shape == "chain" else rng.randint(2, 64)
        most = 9e7 / (vocab * new * (2 if drawn else 1) * (2 if dtype == "float32" else 1))
        batch = max(1, min(_log_int(rng, 1, 64), int(most)))
        return _verify(None, batch, new, vocab, dtype, shape=shape, drawn=drawn, ragged=rng.random() < 0.5,
                       temperature=rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]))
    cube, head_dim = rng.choice([16, 32, 64]), rng.choice([32, 64, 64, 128])
    heads = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24, 32])
    while heads * head_dim > 2048:
        heads //= 2
    page = rng.choice([32, 64, 64, 128, 256])
    groups = rng.choice([1, 1, 1, 2, 3, 5, 8])
    members = max(1, _log_int(rng, 2, 64) // groups)
    mask = rng.choice(["causal", "causal", "tree"])
    new = 1 if rng.random() < 0.5 else rng.randint(2, 64)
    prefix, rest = _log_int(rng, page, 65536), _log_int(rng, 1, 2000)
    c = _share(None, groups, members, rng.choice([0, 0, 1, 5]), new, rng.randint(1, prefix), prefix,
               rng.randint(0, rest), rest, heads, cube, head_dim, page=page, mask=mask, ragged=rng.random() < 0.4,
               scale=rng.choice([cube ** -0.5, 0.25, 0.5, 1.0]))
    # no more work than the largest listed cases: what is read where nothing is shared, scores, matrix work
    while True:
        batch = c["groups"] * c["members"] + c["alone"]
        keys = batch * (c["prefix"] + c["rest_most"] + c["new"])
        if keys * heads * (cube + head_dim) <= 2.5e9 and keys * heads * c["new"] <= 1.2e8 and \
                keys * heads * c["new"] * (cube + head_dim) <= 1.2e10 and work(c)["bytes"] <= 2.2e8:
            return c
        if c["prefix"] > 4 * page:
            c["prefix"] = c["prefix"] * 3 // 4
            c["shortest"] = min(c["shortest"], c["prefix"])
        elif c["new"] > 4:
            c["new"] = c["new"] * 2 // 3
        else:
            c["members"] = max(1, c["members"] * 2 // 3)
            c["rest_most"] = max(1, c["rest_most"] * 3 // 4)
            c["rest_least"] = min(c["rest_least"], c["rest_most"])


def _spread(lo, hi, count, turn):
    """``count`` whole numbers from lo to hi, over their logarithm, in an order without a trend."""
    out = []
    for b in range(count):
        f = (0.5 + 0.6180339887498949 * (b + turn)) % 1.0 if count > 1 else 1.0
        out.append(int(round(math.exp(math.log(lo + 1) + f * (math.log(hi + 1) - math.log(lo + 1))))) - 1)
    return out


def _batch(c):
    return c["groups"] * c["members"] + c["alone"] if c["op"] == "share" else c["batch"]


def _news(c):
    """New tokens of each sequence; some have none where the batch is padded."""
    B = _batch(c)
    return _spread(0, c["new"], B, 3) if c["ragged"] and B > 1 else [c["new"]] * B


def _prefixes(c):
    """Pages of each group's prompt."""
    return [max(1, t // c["page"]) for t in _spread(c["shortest"], c["prefix"], c["groups"], 0)]


def _place(c):
    """The group of each sequence of the batch, -1 for none: members of a group stand apart, as requests come."""
    order = [g for _ in range(c["members"]) for g in range(c["groups"])] + [-1] * c["alone"]
    random.Random(c["groups"] * 1000 + c["members"]).shuffle(order)
    return order


def _lens(c):
    """Tokens of each sequence before the new ones."""
    if c["op"] == "plan":
        return _spread(c["shortest"], c["longest"], c["batch"], 0)
    pages, rest = _prefixes(c), _spread(c["rest_least"], c["rest_most"], _batch(c), 1)
    return [(pages[g] * c["page"] if g >= 0 else 0) + r for g, r in zip(_place(c), rest)]


def _kept(c):
    return [min(k, n) for k, n in zip(_spread(0, c["keep"], c["batch"], 5), _news(c))]


def _parents(c, seed):
    """Of each sequence the parent of each token; -1 for the first, the root."""
    rng = random.Random(seed)
    if c["shape"] == "chain":
        return [list(range(-1, c["new"] - 1))] * c["batch"]
    # three drafts or so of one place, in the order in which a drafter grows its tree
    return [[-1] + [max(0, (i - 1) // 3 - rng.randint(0, 2)) for i in range(1, c["new"])] for _ in range(c["batch"])]


def work(case):
    c = case
    if c["op"] == "share":
        H, m, dv, n, place = c["heads"], c["cube"], c["head_dim"], c["new"], _place(c)
        pages = _prefixes(c)
        own_keys = {"causal": lambda k: k * (k + 1) // 2, "tree": lambda k: k * (k + 1) // 4}[c["mask"]]
        lens, news = _lens(c), _news(c)
        keys = sum(pages) * c["page"] + sum(l + k - (pages[g] * c["page"] if g >= 0 else 0)
                                            for l, k, g in zip(lens, news, place))
        T = len(place) * n
        return {"bytes": 2 * keys * H * (m + dv) + 2 * T * H * (m + dv) + 4 * T * H,
                "flops": 2 * sum(l * k + own_keys(k) for l, k in zip(lens, news)) * H * (m + dv)}
    if c["op"] == "verify":
        size = 4 if c["dtype"] == "float32" else 2
        rows = 0
        for par, k in zip(_parents(c, 0), _news(c)):  # another seed's trees have as many inner places or so
            rows += k + (len({p for p in par[1:k]}) if c["drawn"] and c["temperature"] else 0)
        return {"bytes": rows * c["vocab"] * size + 16 * c["batch"] * c["new"], "flops": 4 * rows * c["vocab"]}
    P, pages = c["page"], 0
    for l, k, kept in zip(_lens(c), _news(c), _kept(c)):
        pages += 2 * (-(-(l + k) // P) - -(-(l + kept) // P))
    return {"bytes": 2 * (24 * c["batch"] + 8 * c["batch"] * c["new"]) + 8 * pages, "flops": 0}


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEVICE)


def _bits(parents):
    """Rows of bits: a token sees its ancestors and itself."""
    rows = []
    for par in parents:
        bits = []
        for i, p in enumerate(par):
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        rows.append([b - (1 << 64) if b >> 63 else b for b in bits])
    return _ints(rows, torch.int64)


def _prepare_share(c, g, rng):
    B, n, H, m, dv, P = _batch(c), c["new"], c["heads"], c["cube"], c["head_dim"], c["page"]
    lens, news, place, pages = _lens(c), _news(c), _place(c), _prefixes(c)
    behind = [-(-(l + n) // P) - (pages[k] if k >= 0 else 0) for l, k in zip(lens, place)]
    pool = sum(pages) + sum(behind) + 1
    order = rng.sample(range(pool), pool - 1)
    take = iter(order)
    prompt = [[next(take) for _ in range(k)] for k in pages]
    rows = [(prompt[k] if k >= 0 else []) + [next(take) for _ in range(r)] for k, r in zip(place, behind)]
    width = max(len(r) for r in rows)
    s = {"table": _ints([r + [-1] * (width - len(r)) for r in rows]), "lens": _ints(lens),
         "new_lens": _ints(news) if c["ragged"] else None, "max_len": max(lens) + n}
    s["codes"] = torch.empty((pool, H, P, m), dtype=torch.float16, device=DEVICE).normal_(generator=g).sigmoid_()
    s["values"] = torch.empty((pool, H, P // 8, dv, 8), dtype=torch.float16, device=DEVICE).normal_(generator=g)
    s["phi"] = torch.sigmoid(torch.randn((B, n, H, m), generator=g, device=DEVICE)).to(torch.float16)
    s["gate_q"] = (1.0 + 0.25 * torch.randn((H, m), generator=g, device=DEVICE)).to(torch.float16)
    s["gate_k"] = (1.0 + 0.25 * torch.randn((H, m), generator=g, device=DEVICE)).to(torch.float16)
    s["tree"] = None
    if c["mask"] == "tree":
        s["tree"] = _bits([[-1] + [rng.randint(max(0, i - 6), i - 1) for i in range(1, n)] for _ in range(B)])
    # which sequences share what, as the program that forked them knows it
    mine = [[b for b in range(B) if place[b] == k] for k in range(c["groups"])]
    s["members"] = _ints([b for k in mine for b in k])
    s["starts"] = _ints([sum(len(k) for k in mine[:i]) for i in range(c["groups"] + 1)])
    s["group"], s["pages"] = _ints(place), _ints(pages)
    s["max_prefix"] = max(pages) * P
    s["max_rest"] = max(l + n - (pages[k] * P if k >= 0 else 0) for l, k in zip(lens, place))
    return s


def _prepare_verify(c, g, seed):
    B, n, V, dtype = c["batch"], c["new"], c["vocab"], _TYPES[c["dtype"]]
    parents = _parents(c, seed)
    par = _ints(parents, torch.int64)
    # a drafter that is right more often than not: the target's logits and the drafter's have most in common
    base = torch.randn((B, n, V), generator=g, device=DEVICE).mul_(2.5)
    s = {"logits": (base + 0.5 * torch.randn((B, n, V), generator=g, device=DEVICE)).to(dtype)}
    draft = (base + 0.5 * torch.randn((B, n, V), generator=g, device=DEVICE)).to(dtype)
    del base
    tokens = torch.randint(0, V, (B, n), generator=g, device=DEVICE)
    if n > 1 and c["drawn"]:
        T = c["temperature"] or 1.0
        for i in range(1, n):
            row = draft[torch.arange(B, device=DEVICE), par[:, i]].float() / T
            tokens[:, i] = torch.multinomial(torch.softmax(row, -1), 1, generator=g)[:, 0]
    elif n > 1:
        best = draft.topk(min(V, n), -1).indices
        turn = _ints([[sum(q == p for q in row[:i]) for i, p in enumerate(row)] for row in parents], torch.int64)
        at = torch.arange(B, device=DEVICE)[:, None]
        tokens[:, 1:] = best[at, par[:, 1:], turn[:, 1:].clamp(max=best.shape[-1] - 1)]
    s["tokens"] = tokens
    s["draft_logits"] = draft[:, : n - 1].contiguous() if c["drawn"] and n > 1 else None
    s["uniform"] = torch.rand((B, n), generator=g, device=DEVICE)
    s["tree"] = _bits(parents) if c["shape"] == "tree" else None
    s["new_lens"] = _ints(_news(c)) if c["ragged"] else None
    return s


def _prepare_plan(c, rng):
    P, lens, news = c["page"], _lens(c), _news(c)
    have = [-(-l // P) for l in lens]
    width = max(-(-(l + c["new"]) // P) for l in lens)
    asked = sum(-(-(l + k) // P) - h for l, k, h in zip(lens, news, have))
    spare = asked * c["spare"] // 100
    pool = sum(have) + spare
    order = rng.sample(range(pool), pool)
    take = iter(order)
    rows = [[next(take) for _ in range(h)] + [-1] * (width - h) for h in have]
    free = list(take) + [-1] * (asked + 1)  # the stack has room for more than there is
    return {"table": _ints(rows), "held": _ints(have), "lens": _ints(lens), "new_lens": _ints(news),
            "kept": _ints(_kept(c)), "free": _ints(free), "free_count": _ints([spare])}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    s = {"share": lambda: _prepare_share(case, g, rng), "verify": lambda: _prepare_verify(case, g, seed),
         "plan": lambda: _prepare_plan(case, rng)}[case["op"]]()
    s["case"] = dict(case)
    return s


def run(state):
    if own:
        return _run_own(state)
    return {"share": _plain_share, "verify": _plain_verify, "plan": _plain_plan}[state["case"]["op"]](state)


def _run_own(s):
    import morphottention_amd as ma
    c = s["case"]
    if c["op"] == "share":
        shared = ma.SharedPrefix(s["members"], s["starts"], s["group"], s["pages"], max_prefix=s["max_prefix"],
                                 max_rest=s["max_rest"])
        out, lse = ma.morpho_cache_attention(s["phi"], s["gate_q"], s["gate_k"], s["codes"], s["values"], s["table"],
                                             s["lens"], new_lens=s["new_lens"], tree=s["tree"], scale=c["scale"],
                                             max_len=s["max_len"], shared=shared)
        return {"out": out, "lse": lse}
    if c["op"] == "verify":
        keep, keep_lens, token = ma.morpho_verify_drafts(s["logits"], s["tokens"], s["uniform"], tree=s["tree"],
                                                         new_lens=s["new_lens"], draft_logits=s["draft_logits"],
                                                         temperature=c["temperature"])
        return {"keep": keep, "keep_lens": keep_lens, "token": token}
    out = {}
    for at, news in (("", s["new_lens"]), ("_kept", s["kept"])):
        out["granted" + at], out["slots" + at] = ma.morpho_cache_plan(
            s["table"], s["held"], s["lens"], s["free"], s["free_count"], c["new"], new_lens=news, page_size=c["page"])
    return out | {k: s[k] for k in ("table", "held", "free", "free_count")}


# ---------------------------------------------------------------- plain forms
def _plain_share(s):
    """Attention of every sequence over its own pages."""
    c = s["case"]
    H, m, dv, P, n = c["heads"], c["cube"], c["head_dim"], c["page"], c["new"]
    B = s["phi"].shape[0]
    used = (s["max_len"] + P - 1) // P
    table = s["table"][:, :used].long().clamp(min=0)
    L = table.shape[1] * P
    k = s["codes"][table].permute(0, 2, 1, 3, 4).float().reshape(B, H, L, m)
    v = s["values"][table].permute(0, 2, 1, 3, 5, 4).float().reshape(B, H, L, dv)
    phi = s["phi"].float().transpose(1, 2)
    gate = (s["gate_q"].float() * s["gate_k"].float())[None, :, None, :]
    u = c["scale"] * gate * (2.0 * phi - 1.0)
    row = c["scale"] * (gate * phi).sum(-1, keepdim=True)
    sc = torch.matmul(u, k.transpose(2, 3).contiguous()) - row
    lens = s["lens"].long()[:, None, None]
    new = torch.full_like(lens, n) if s["new_lens"] is None else s["new_lens"].long()[:, None, None]
    j = torch.arange(L, device=k.device)[None, None, :]
    i = torch.arange(n, device=k.device)[None, :, None]
    seen = (j < lens + new) & (i < new)
    if c["mask"] == "tree":
        bit = (s["tree"][:, :, None] >> (j - lens).clamp(0, 63)) & 1
        seen = seen & ((j < lens) | (bit == 1))
    else:
        seen = seen & (j <= lens + i)
    sc = sc.masked_fill(~seen[:, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    some = top > -math.inf
    top = torch.where(some, top, torch.zeros_like(top))
    p = torch.exp(sc - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(some, total, torch.ones_like(total))
    lse = torch.where(some, top * math.log2(math.e) + torch.log2(total), torch.full_like(top, _NONE))
    return {"out": out.transpose(1, 2).reshape(B, n, H * dv).to(torch.float16), "lse": lse.reshape(B * H, n)}


def _softmax64(x, temperature):
    x = x.double() / temperature
    w = torch.exp(x - x.amax(-1, keepdim=True))
    return w / w.sum(-1, keepdim=True)


def _plain_verify(s):
    """In 64 bits: what is decided are whole numbers, next to borders."""
    c = s["case"]
    tokens, tree, draft = s["tokens"], s["tree"], s["draft_logits"]
    B, n, V = s["logits"].shape
    at, place = torch.arange(B, device=tokens.device), torch.arange(n, device=tokens.device)
    new = torch.full((B,), n, device=tokens.device) if s["new_lens"] is None else s["new_lens"].long()
    if tree is None:
        parent = (place - 1).expand(B, n)
    else:  # the highest bit below a token's own
        below = ((tree[:, :, None] >> place) & 1).bool() & (place < place[:, None])
        parent = torch.where(below, place, torch.full_like(place, -1)).amax(-1)
    node = torch.zeros_like(new)
    taken = place.expand(B, n) == 0
    if not c["temperature"]:
        best = s["logits"].float().argmax(-1)
        for i in range(1, n):
            ok = (parent[:, i] == node) & (tokens[:, i] == best[at, node]) & (i < new)
            node = torch.where(ok, i, node)
            taken = taken | (ok[:, None] & (place == i))
        token = best[at, node]
    else:
        p = _softmax64(s["logits"], c["temperature"])
        q = None if draft is None else _softmax64(draft, c["temperature"])
        u = s["uniform"].double()
        left = p[:, 0]  # what is left of the distribution at the token at hand, and its sum
        for i in range(1, n):
            mine = (parent[:, i] == node) & (i < new)
            t = tokens[:, i: i + 1]
            if q is None:
                guess = torch.zeros_like(left).scatter_(1, t, 1.0)
                minus = torch.where(guess > 0, torch.zeros_like(left), left)
            else:
                guess = q[at, parent[:, i].clamp(min=0)]
                minus = (left / left.sum(-1, keepdim=True) - guess).clamp(min=0.0)
            ok = mine & (u[:, i] * (guess.gather(1, t) * left.sum(-1, keepdim=True))[:, 0] < left.gather(1, t)[:, 0])
            left = torch.where(ok[:, None], p[:, i], torch.where(mine[:, None], minus, left))
            node = torch.where(ok, i, node)
            taken = taken | (ok[:, None] & (place == i))
        run_sum = left.cumsum(-1)
        token = (run_sum <= u[:, :1] * run_sum[:, -1:]).sum(-1).clamp(max=V - 1)
    taken = taken & (place < new[:, None])
    count = taken.sum(-1)
    rank = torch.where(taken, taken.cumsum(-1) - 1, torch.full_like(parent, n))
    keep = torch.full((B, n + 1), -1, dtype=torch.int32, device=tokens.device)
    keep.scatter_(1, rank, torch.where(taken, place.expand(B, n), torch.full_like(parent, -1)).to(torch.int32))
    keep[:, n] = -1
    return {"keep": keep[:, :n].contiguous(), "keep_lens": count.to(torch.int32),
            "token": torch.where(new > 0, token, torch.full_like(token, -1))}


def _plain_step(s, news):
    c = s["case"]
    P, table, free = c["page"], s["table"], s["free"]
    B, W = table.shape
    col = torch.arange(W, device=table.device)[None, :]
    lens, held = s["lens"].long()[:, None], s["held"].long()[:, None]
    new = news.long()[:, None]
    want = (lens + new + P - 1) // P
    fits = want <= W
    back = fits & (col >= want) & (col < held)
    count = s["free_count"].long()
    turn = back.flatten().long().cumsum(0).view(B, W)
    total = turn[-1, -1]
    F = free.shape[0]
    spot = torch.where(back, count + total - turn, torch.full_like(turn, F))
    stack = torch.cat((free, free.new_zeros(1))).scatter(0, spot.flatten(), table.flatten())[:F]
    count = count + total
    need = torch.where(fits, (want - held).clamp(min=0), torch.zeros_like(want))
    upto = need.cumsum(0)
    ok = fits & ((need == 0) | (upto <= count))
    more = ok & (col >= held) & (col < want)
    got = stack.long()[(count - 1 - (upto - need + col - held)).clamp(0, F - 1)]
    rows = torch.where(more, got, torch.where(back, torch.full_like(got, -1), table.long()))
    granted = torch.where(ok, new, torch.zeros_like(new))
    i = torch.arange(c["new"], device=table.device)[None, :]
    pos = lens + i
    page = rows.gather(1, (pos // P).clamp(max=W - 1))
    slots = torch.where((i < granted) & (page >= 0), page * P + pos % P, torch.full_like(page, -1))
    table.copy_(rows)
    free.copy_(stack)
    s["held"].copy_(torch.where(ok, want, held)[:, 0])
    s["free_count"].copy_(count - torch.where(ok, need, torch.zeros_like(need)).sum())
    return granted[:, 0].to(torch.int32), slots


def _plain_plan(s):
    granted, slots = _plain_step(s, s["new_lens"])
    granted_kept, slots_kept = _plain_step(s, s["kept"])
    return {"granted": granted, "slots": slots, "granted_kept": granted_kept, "slots_kept": slots_kept} | \
        {k: s[k] for k in ("table", "held", "free", "free_count")}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"share": _exact_share, "verify": _exact_verify, "plan": lambda c, s: None}[case["op"]](case, s)


def _exact_share(c, s):
    H, m, dv, P, n, B = c["heads"], c["cube"], c["head_dim"], c["page"], c["new"], _batch(c)
    lens, news = _lens(c), _news(c)
    out = torch.zeros((B, n, H, dv), dtype=torch.float64, device=DEVICE)
    lse = torch.full((B, H, n), _NONE, dtype=torch.float64, device=DEVICE)
    gate = s["gate_q"].double() * s["gate_k"].double()
    for b in range(B):
        total = lens[b] + news[b]
        if not news[b]:
            continue
        mine = s["table"][b, : (total + P - 1) // P].long()
        for h in range(H):
            key = s["codes"][mine, h].double().reshape(-1, m)[:total]
            val = s["values"][mine, h].double().transpose(2, 3).reshape(-1, dv)[:total]
            q = s["phi"][b, : news[b], h].double()
            sc = 2.0 * torch.matmul(q * gate[h], key.T.contiguous()) - (q @ gate[h])[:, None] - (key @ gate[h])[None, :]
            seen = torch.ones_like(sc, dtype=torch.bool)
            if c["mask"] == "causal":
                seen = torch.tril(seen, diagonal=lens[b])
            else:
                k = torch.arange(news[b], device=sc.device)
                seen[:, lens[b]:] = ((s["tree"][b, : news[b], None] >> k) & 1).bool()
            sc = (c["scale"] * sc).masked_fill(~seen, -math.inf)
            part = torch.logsumexp(sc, dim=1)
            out[b, : news[b], h] = torch.matmul(torch.exp(sc - part[:, None]), val)
            lse[b, h, : news[b]] = part / math.log(2.0)
    return {"out": out.reshape(B, n, H * dv), "lse": lse.reshape(B * H, n)}


def _exact_verify(c, s):
    """One sequence after another, as the rule is told: walk down from the root, ask its drafts in order."""
    import numpy as np
    n, T = c["new"], c["temperature"]
    news = _news(c)
    tokens, u = s["tokens"].tolist(), s["uniform"].tolist()
    rows = s["tree"].tolist() if s["tree"] is not None else None

    def dist(row):
        x = row.double().cpu().numpy() / T
        x = np.exp(x - x.max())
        return x / x.sum()
    keep, count, token = [], [], []
    for b in range(c["batch"]):
        if not news[b]:
            keep.append([-1] * n)
            count.append(0)
            token.append(-1)
            continue
        parent = [i - 1 for i in range(n)] if rows is None else \
            [max([k for k in range(i) if rows[b][i] >> k & 1], default=-1) for i in range(n)]
        path = [0]
        while True:
            node, down = path[-1], None
            children = [i for i in range(1, news[b]) if parent[i] == node]
            if not T:
                last = int(s["logits"][b, node].float().cpu().numpy().argmax())
                down = next((i for i in children if tokens[b][i] == last), None)
            else:
                r = dist(s["logits"][b, node])
                q = dist(s["draft_logits"][b, node]) if children and s["draft_logits"] is not None else None
                for i in children:
                    t = tokens[b][i]
                    if u[b][i] * (1.0 if q is None else q[t]) < r[t]:
                        down = i
                        break
                    if q is None:
                        r[t] = 0.0
                    else:
                        r = np.maximum(r - q, 0.0)
                    r = r / r.sum()
                if down is None:
                    last = int(np.searchsorted(np.cumsum(r), u[b][0] * r.sum(), side="right"))
            if down is None:
                break
            path.append(down)
        keep.append(path + [-1] * (n - len(path)))
        count.append(len(path))
        token.append(min(last, c["vocab"] - 1))
    return {"keep": _ints(keep), "keep_lens": _ints(count), "token": _ints(token, torch.int64)}
