"""What the cache operators' speed is judged on: serving a causal ``MorphoAttention`` from a
paged cache, one operator a case, from one token of one user to long contexts and prompts.

A case is a dict of plain values:

* ``op``: ``append`` (``morpho_cache_append``), ``attend`` (``morpho_cache_attention``),
  ``copy`` (``morpho_cache_copy_pages``) or ``compact`` (``morpho_cache_compact``);
* ``batch`` sequences of ``new`` tokens each (fewer where ``ragged``), after contexts of
  ``shortest`` to ``longest`` tokens; ``heads``, ``cube`` (codes per head), ``head_dim``
  (value columns per head), ``page`` (tokens a page), ``layers``;
* ``mask``: ``causal``, ``full`` or ``tree`` (the new tokens are drafts that see their
  ancestors), ``mask_diag``, ``scale``, ``projection``;
* ``pages``: the pairs of a copy; ``keep``: the tokens that a compaction keeps at most.

The cache's layout (every tensor float16, as everywhere in the framework):

* ``codes`` [layers, pages, H, page, cube], the key codes phi;
* ``values`` [layers, pages, H, page / 8, head_dim, 8], eight tokens of a column together;
* ``table`` [batch, pages a sequence] int32, ``lens`` [batch] int32, the tokens before the new ones.
"""

from __future__ import annotations

import math
import random

import torch

DEVICE = "cuda"

# set by the harness: the framework's kernels instead of the plain forms
own = False


def _case(name, op, batch, new, shortest, longest, heads, cube, head_dim, *, page=64, layers=1, mask="causal",
          mask_diag=False, ragged=False, scale=1.0, projection="sigmoid", pages=0, keep=0):
    c = {"op": op, "batch": batch, "new": new, "shortest": shortest, "longest": longest, "heads": heads, "cube": cube,
         "head_dim": head_dim, "page": page, "layers": layers, "mask": mask, "mask_diag": mask_diag, "ragged": ragged,
         "scale": scale, "projection": projection, "pages": pages, "keep": keep}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the next token of one user through the smallest module of the tests: a launch and its latency
        _case("append_one", "append", 1, 1, 37, 37, 8, 16, 32),
        # the next token of 64 users through the headline module
        _case("append_batch", "append", 64, 1, 0, 250, 16, 16, 64),
        # drafted tokens of 16 users through the widest module, not as many for each
        _case("append_drafts", "append", 16, 12, 0, 200, 32, 64, 64, ragged=True),
        # prompts of different lengths, behind a short common prefix
        _case("append_prompt", "append", 3, 3001, 5, 90, 16, 32, 64, ragged=True),
        # the next token of one user early in a conversation
        _case("attend_one", "attend", 1, 1, 99, 99, 8, 16, 32),
        # the next token of 64 users, contexts from a few tokens to thousands
        _case("attend_batch", "attend", 64, 1, 1, 8191, 16, 16, 64),
        # the next token of one user after a very long context
        _case("attend_long", "attend", 1, 1, 131070, 131070, 16, 32, 64, scale=0.5),
        # a tree of drafts for each of 16 users of the widest module
        _case("attend_tree", "attend", 16, 48, 300, 4000, 32, 64, 64, mask="tree", ragged=True, scale=0.125),
        # a piece of a prompt that is taken in pieces, behind what is there already
        _case("attend_chunk", "attend", 4, 1000, 3000, 4096, 16, 16, 64),
        # a fork's copies on write: the last pages of a few sequences, in all layers
        _case("copy_fork", "copy", 1, 1, 0, 0, 16, 16, 64, layers=12, pages=5),
        # the prefixes of a beam search's survivors copied into pages of their own
        _case("copy_beams", "copy", 1, 1, 0, 0, 16, 32, 64, layers=2, pages=700),
        # the accepted path of each user's tree moves to the front of the drafts, in all layers
        _case("compact_accept", "compact", 32, 48, 20, 500, 16, 16, 64, layers=12, keep=9, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "copy", "compact"])
    cube, head_dim = rng.choice([16, 32, 64]), rng.choice([32, 64, 64, 128])
    heads = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24, 32])
    while heads * head_dim > 2048:
        heads //= 2
    page = rng.choice([32, 64, 64, 128, 256])
    scale = rng.choice([cube ** -0.5, 0.25, 0.5, 1.0])
    ragged = rng.random() < 0.5
    if op == "append":
        batch = _log_int(rng, 1, 64)
        new = max(1, _log_int(rng, 1, 4000) // batch) if rng.random() < 0.6 else 1
        longest = rng.randint(0, 300)
        return _case(None, op, batch, new, rng.randint(0, longest), longest, heads, cube, head_dim, page=page,
                     ragged=ragged, projection=rng.choice(["sigmoid", "sigmoid", "hardtanh01", "identity"]))
    if op == "attend":
        mask = rng.choice(["causal", "causal", "tree", "full"])
        batch, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 100000)
        new = 1 if rng.random() < 0.4 else rng.randint(2, 64) if mask == "tree" else _log_int(rng, 2, 900)
        shortest = rng.randint(0, longest)
        c = _case(None, op, batch, new, shortest, longest, heads, cube, head_dim, page=page, mask=mask,
                  mask_diag=mask != "tree" and rng.random() < 0.2, ragged=ragged, scale=scale)
        # no more work than the largest listed cases: matrix work, bytes and values of the scores
        while _pairs(c) * heads * (cube + head_dim) > 2.2e10 or \
                batch * (longest + new) * heads * (cube + head_dim) > 6e8 or batch * heads * new * (longest + new) > 3e8:
            if c["batch"] > 1:
                c["batch"] = batch = batch * 2 // 3
            elif c["new"] > 64:
                c["new"] = new = new * 2 // 3
            else:
                c["longest"] = longest = longest * 3 // 4
                c["shortest"] = min(shortest, longest)
        return c
    layers = rng.choice([1, 2, 4, 12])
    if op == "copy":
        most = int(2.5e8 / (layers * heads * page * (cube + head_dim) * 2))
        return _case(None, op, 1, 1, 0, 0, heads, cube, head_dim, page=page, layers=layers,
                     pages=_log_int(rng, 1, max(2, min(2000, most))))
    batch = _log_int(rng, 1, 32)
    most = int(6e7 / (layers * heads * (cube + head_dim) * batch))
    new = min(_log_int(rng, 2, 4000), max(2, most))
    longest = min(rng.randint(0, 300), most)
    return _case(None, op, batch, new, rng.randint(0, longest), longest, heads, cube, head_dim, page=page,
                 layers=layers, ragged=ragged, keep=rng.randint(1, new))


def _spread(lo, hi, count, turn):
    """``count`` whole numbers from lo to hi, over their logarithm, in an order without a trend."""
    out = []
    for b in range(count):
        f = (0.5 + 0.6180339887498949 * (b + turn)) % 1.0 if count > 1 else 1.0
        out.append(int(round(math.exp(math.log(lo + 1) + f * (math.log(hi + 1) - math.log(lo + 1))))) - 1)
    return out


def _lens(c):
    return _spread(c["shortest"], c["longest"], c["batch"], 0)


def _news(c):
    """New tokens of each sequence; some have none where the batch is padded."""
    most = c["new"]
    return _spread(0, most, c["batch"], 3) if c["ragged"] and c["batch"] > 1 else [most] * c["batch"]


def _keeps(c):
    return [min(k, n) for k, n in zip(_spread(0, c["keep"], c["batch"], 5) if c["ragged"] and c["batch"] > 1
                                      else [c["keep"]] * c["batch"], [c["new"]] * c["batch"])]


def _context(c):
    return sum(l + n for l, n in zip(_lens(c), _news(c)))


def _pairs(c):
    """(query, key) pairs of a head; a drafted token is taken to see half of the drafts before it."""
    own_keys = {"causal": lambda n: n * (n + 1) // 2, "full": lambda n: n * n, "tree": lambda n: n * (n + 1) // 4}
    return sum(l * n + own_keys[c["mask"]](n) for l, n in zip(_lens(c), _news(c)))


def work(case):
    c = case
    H, m, dv, D = c["heads"], c["cube"], c["head_dim"], c["heads"] * c["head_dim"]
    if c["op"] == "append":
        T, stored, C = c["batch"] * c["new"], sum(_news(c)), H * (m + dv)
        return {"bytes": 2 * (T * D + C * D + T * H * m + stored * C), "flops": 2 * T * D * C}
    if c["op"] == "attend":
        T = c["batch"] * c["new"]
        return {"bytes": 2 * _context(c) * H * (m + dv) + 2 * T * H * (m + dv) + 4 * T * H,
                "flops": 2 * _pairs(c) * H * (m + dv)}
    if c["op"] == "copy":
        return {"bytes": 4 * c["layers"] * c["pages"] * H * c["page"] * (m + dv), "flops": 0}
    return {"bytes": 4 * c["layers"] * sum(_keeps(c)) * H * (m + dv), "flops": 0}


def _normal(shape, g, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * scale).to(torch.float16)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    B, n, H, m, dv, P, L = (c[k] for k in ("batch", "new", "heads", "cube", "head_dim", "page", "layers"))
    D = H * dv
    lens = _lens(c)
    if c["op"] == "copy":
        per, pool = 0, 2 * c["pages"] + 3
    else:
        per = (max(lens) + n + P - 1) // P
        pool = B * per + 1
    s = {"case": dict(c)}
    # float16 normal values are drawn a layer and a share of the pages at a time: the pools are large
    s["codes"] = torch.empty((L, pool, H, P, m), dtype=torch.float16, device=DEVICE)
    s["values"] = torch.empty((L, pool, H, P // 8, dv, 8), dtype=torch.float16, device=DEVICE)
    for l in range(L):
        s["codes"][l].normal_(generator=g).sigmoid_()
        s["values"][l].normal_(generator=g)
    if c["op"] == "copy":
        order = rng.sample(range(pool), 2 * c["pages"])
        s["src"] = torch.tensor(order[: c["pages"]], dtype=torch.int32, device=DEVICE)
        s["dst"] = torch.tensor(order[c["pages"]:], dtype=torch.int32, device=DEVICE)
        return s
    s["table"] = torch.tensor(rng.sample(range(pool), B * per), dtype=torch.int32, device=DEVICE).view(B, per)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    if c["op"] == "compact":
        kept = _keeps(c)
        rows = [sorted(rng.sample(range(n), k)) + [0] * (max(1, c["keep"]) - k) for k in kept]
        s["keep"] = torch.tensor(rows, dtype=torch.int32, device=DEVICE)
        s["keep_lens"] = torch.tensor(kept, dtype=torch.int32, device=DEVICE)
        return s
    s["new_lens"] = torch.tensor(_news(c), dtype=torch.int32, device=DEVICE) if c["ragged"] else None
    s["max_len"] = max(lens) + n  # the host's own count of the tokens it has handed in
    if c["op"] == "append":
        s["x"] = _normal((B, n, D), g)
        # [W_phi | W_V] transposed, as a program keeps it from its start on
        s["weights"] = _normal((H * m + D, D), g, D ** -0.5)
    else:
        s["phi"] = torch.sigmoid(torch.randn((B, n, H, m), generator=g, device=DEVICE)).to(torch.float16)
        s["gate_q"] = (1.0 + 0.25 * torch.randn((H, m), generator=g, device=DEVICE)).to(torch.float16)
        s["gate_k"] = (1.0 + 0.25 * torch.randn((H, m), generator=g, device=DEVICE)).to(torch.float16)
        s["tree"] = None
        if c["mask"] == "tree":
            rows = []
            for _ in range(B):
                bits = []
                for k in range(n):
                    parent = rng.randint(max(-1, k - 6), k - 1)
                    bits.append((bits[parent] if parent >= 0 else 0) | 1 << k)
                rows.append([b - (1 << 64) if b >> 63 else b for b in bits])
            s["tree"] = torch.tensor(rows, dtype=torch.int64, device=DEVICE)
    return s


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "copy": _plain_copy,
            "compact": _plain_compact}[state["case"]["op"]](state)


def _run_own(s):
    import morphottention_amd as ma
    c = s["case"]
    if c["op"] == "append":
        phi = ma.morpho_cache_append(s["x"], s["weights"], s["codes"][0], s["values"][0], s["table"], s["lens"],
                                     new_lens=s["new_lens"], projection=c["projection"])
        return {"phi": phi, "codes": s["codes"], "values": s["values"]}
    if c["op"] == "attend":
        out, lse = ma.morpho_cache_attention(s["phi"], s["gate_q"], s["gate_k"], s["codes"][0], s["values"][0],
                                             s["table"], s["lens"], new_lens=s["new_lens"], tree=s["tree"],
                                             scale=c["scale"], causal=c["mask"] != "full", mask_diag=c["mask_diag"],
                                             max_len=s["max_len"])
        return {"out": out, "lse": lse}
    if c["op"] == "copy":
        ma.morpho_cache_copy_pages(s["codes"], s["values"], s["src"], s["dst"])
    else:
        ma.morpho_cache_compact(s["codes"], s["values"], s["table"], s["lens"], s["keep"], keep_lens=s["keep_lens"])
    return {"codes": s["codes"], "values": s["values"]}


# ---------------------------------------------------------------- plain forms
def _project(z, projection):
    if projection == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    return ((z + 1.0) * 0.5).clamp(0.0, 1.0) if projection == "hardtanh01" else z


def _slots(table, pos, page):
    """Page and place of positions [B, k]; positions behind the table's end take its last page."""
    at = (pos // page).clamp(max=table.shape[1] - 1).long()
    return table.long().gather(1, at), (pos % page).long()


def _plain_append(s):
    c = s["case"]
    H, m, dv, P, n = c["heads"], c["cube"], c["head_dim"], c["page"], c["new"]
    x = s["x"]
    B = x.shape[0]
    z = x.float() @ s["weights"].float().t()
    phi = _project(z[..., : H * m], c["projection"]).to(torch.float16).view(B, n, H, m)
    v = z[..., H * m:].to(torch.float16).view(B, n, H, dv)
    codes, values = s["codes"][0], s["values"][0]
    i = torch.arange(n, device=x.device)
    page, slot = _slots(s["table"], s["lens"][:, None] + i, P)
    # a padding row stores what is there already
    real = None if s["new_lens"] is None else (i < s["new_lens"][:, None])[:, :, None, None]
    codes[page, :, slot] = phi if real is None else torch.where(real, phi, codes[page, :, slot])
    values[page, :, slot // 8, :, slot % 8] = v if real is None else \
        torch.where(real, v, values[page, :, slot // 8, :, slot % 8])
    return {"phi": phi, "codes": s["codes"], "values": s["values"]}


def _plain_attend(s):
    c = s["case"]
    H, m, dv, P, n = c["heads"], c["cube"], c["head_dim"], c["page"], c["new"]
    B = s["phi"].shape[0]
    used = (s["max_len"] + P - 1) // P
    table = s["table"][:, :used].long()
    L = used * P
    k = s["codes"][0][table].permute(0, 2, 1, 3, 4).float().reshape(B, H, L, m)
    v = s["values"][0][table].permute(0, 2, 1, 3, 5, 4).float().reshape(B, H, L, dv)
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
    elif c["mask"] == "causal":
        seen = seen & (j <= lens + i)
    if c["mask_diag"]:
        seen = seen & (j != lens + i)
    seen = seen[:, None]
    sc = sc.masked_fill(~seen, -math.inf)
    top = sc.amax(-1, keepdim=True)
    some = top > -math.inf
    top = torch.where(some, top, torch.zeros_like(top))
    p = torch.exp(sc - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(some, total, torch.ones_like(total))
    lse = torch.where(some, top * math.log2(math.e) + torch.log2(total), torch.full_like(top, -torch.finfo(torch.float32).max))
    return {"out": out.transpose(1, 2).reshape(B, n, H * dv).to(torch.float16), "lse": lse.reshape(B * H, n)}


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["codes"][:, dst] = s["codes"][:, src]
    s["values"][:, dst] = s["values"][:, src]
    return {"codes": s["codes"], "values": s["values"]}


def _plain_compact(s):
    P = s["case"]["page"]
    codes, values = s["codes"], s["values"]
    i = torch.arange(s["keep"].shape[1], device=codes.device)
    real = i < s["keep_lens"][:, None]
    to = s["lens"][:, None] + i
    page, slot = _slots(s["table"], to, P)
    was, place = _slots(s["table"], torch.where(real, s["lens"][:, None] + s["keep"], to), P)
    k, v = codes[:, was, :, place], values[:, was, :, place // 8, :, place % 8]
    codes[:, page, :, slot] = k
    values[:, page, :, slot // 8, :, slot % 8] = v
    return {"codes": codes, "values": values}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    H, m, dv, P = c["heads"], c["cube"], c["head_dim"], c["page"]
    codes, values = s["codes"], s["values"]
    if c["op"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            codes[:, b].copy_(codes[:, a])
            values[:, b].copy_(values[:, a])
        return {"codes": codes, "values": values}
    table, lens = s["table"].tolist(), _lens(c)
    if c["op"] == "compact":
        for b, count in enumerate(_keeps(c)):
            for i, k in enumerate(s["keep"][b, :count].tolist()):  # ascending: nothing is overwritten before it moves
                a, z = lens[b] + k, lens[b] + i
                if a != z:
                    codes[:, table[b][z // P], :, z % P] = codes[:, table[b][a // P], :, a % P]
                    values[:, table[b][z // P], :, z % P // 8, :, z % 8] = \
                        values[:, table[b][a // P], :, a % P // 8, :, a % 8]
        return {"codes": codes, "values": values}
    news = _news(c)
    if c["op"] == "append":
        codes, values = codes.double(), values.double()
        B, n = c["batch"], c["new"]
        w = s["weights"].double()
        phis = torch.empty((B, n, H, m), dtype=torch.float64, device=codes.device)
        for b in range(B):
            x = s["x"][b].double()
            z = torch.matmul(x, w[: H * m].T.contiguous())
            phi = {"sigmoid": torch.sigmoid, "identity": lambda t: t,
                   "hardtanh01": lambda t: torch.clamp(t / 2 + 0.5, 0, 1)}[c["projection"]](z).reshape(n, H, m)
            v = torch.matmul(x, w[H * m:].T.contiguous()).reshape(n, H, dv)
            phis[b] = phi
            i = 0
            while i < news[b]:  # a page, or what is left of one, at a time
                at = lens[b] + i
                k = min(P - at % P, news[b] - i)
                codes[0, table[b][at // P], :, at % P: at % P + k] = phi[i: i + k].transpose(0, 1)
                rows = torch.arange(at % P, at % P + k, device=codes.device)
                values[0, table[b][at // P]][:, rows // 8, :, rows % 8] = v[i: i + k]
                i += k
        return {"phi": phis, "codes": codes, "values": values}
    B, n = c["batch"], c["new"]
    out = torch.zeros((B, n, H, dv), dtype=torch.float64, device=codes.device)
    lse = torch.full((B, H, n), -torch.finfo(torch.float32).max, dtype=torch.float64, device=codes.device)
    gate = s["gate_q"].double() * s["gate_k"].double()
    for b in range(B):
        total = lens[b] + news[b]
        if not news[b]:
            continue
        mine = s["table"][b, : (total + P - 1) // P].long()
        for h in range(H):
            key = codes[0, mine, h].double().reshape(-1, m)[:total]
            val = values[0, mine, h].double().transpose(2, 3).reshape(-1, dv)[:total]
            q = s["phi"][b, : news[b], h].double()
            sc = 2.0 * torch.matmul(q * gate[h], key.T.contiguous()) - (q @ gate[h])[:, None] - (key @ gate[h])[None, :]
            sc = c["scale"] * sc
            seen = torch.ones_like(sc, dtype=torch.bool)
            if c["mask"] == "causal":
                seen = torch.tril(seen, diagonal=lens[b])
            elif c["mask"] == "tree":
                k = torch.arange(news[b], device=sc.device)
                seen[:, lens[b]:] = ((s["tree"][b, : news[b], None] >> k) & 1).bool()
            if c["mask_diag"]:
                i = torch.arange(news[b], device=sc.device)
                seen[i, lens[b] + i] = False
            sc = sc.masked_fill(~seen, -math.inf)
            part = torch.logsumexp(sc, dim=1)
            some = part > -math.inf
            weight = torch.where(some[:, None], torch.exp(sc - part[:, None]), torch.zeros_like(sc))
            out[b, : news[b], h] = torch.matmul(weight, val)
            lse[b, h, : news[b]] = torch.where(some, part / math.log(2.0), lse[b, h, : news[b]])
    return {"out": out.reshape(B, n, H * dv), "lse": lse.reshape(B * H, n)}
