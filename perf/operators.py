"""A paged KV cache: its bookkeeping (`reserve`, `free`, `fork`, `compact`), `rope_append`, which writes a layer's new tokens into its pages,
and `attention`, which reads them and multiplies a prefix that several sequences share out once for all of them.

The cache is `models.pages.PagedCache`: pool fp16 [layers, 2 (K, V), pages, KV heads, page, 128]; table int32 [slots, pages of a slot], -1
where there is none; lengths int32 [slots]; refs int32 [pages], how many slots hold a page; the last three lie in one tensor, `book`.
"""
import math
import os
import random
import sys

import torch

own = False

PKG = os.path.join(os.getcwd(), "sbvr-cpu-arm_b200")      # the package's folder name is not an importable name
D = 128
THETA = 500000.0

# query heads, KV heads of this repository's presets, and three head layouts of no preset
HEADS = {"tiny": (4, 2), "tiny8": (16, 8), "8b": (32, 8), "70b": (64, 8), "equal": (8, 8), "single": (8, 1), "odd": (15, 3)}


def listed():
    return [
        # Four users of the tiny preset on a short common instruction, one token each: latency only.
        {"name": "attention_small", "kind": "attention", "heads": "tiny", "page": 16, "groups": 1, "per": 4, "shared": 256, "own": 40, "new": 1},
        # Four documents, sixteen questions to each, an 8B layer, one token per question.
        {"name": "attention_documents", "kind": "attention", "heads": "8b", "page": 64, "groups": 4, "per": 16, "shared": 8000, "own": 600, "new": 1},
        # 128 samples on one very long prompt, the largest call there is.
        {"name": "attention_long", "kind": "attention", "heads": "8b", "page": 64, "groups": 1, "per": 128, "shared": 65536, "own": 900, "new": 1},
        # The questions themselves: eight prompts of up to 300 tokens behind a common text of an odd length.
        {"name": "attention_prompts", "kind": "attention", "heads": "8b", "page": 32, "groups": 1, "per": 8, "shared": 4001, "own": 300, "new": 300},
        # A decode step's rotary embedding and append, 64 users.
        {"name": "append_step", "kind": "append", "heads": "8b", "page": 64, "seqs": 64, "before": 70, "new": 1},
        # Prompts of 16 users, of uneven lengths, behind what their slots hold.
        {"name": "append_prompts", "kind": "append", "heads": "8b", "page": 16, "seqs": 16, "before": 33, "new": 500},
        # Beam search, eight beams in slots of their own: every beam goes on from one of them.
        {"name": "fork_beams", "kind": "fork", "layers": 2, "heads": "tiny", "page": 16, "slots": 8, "children": 8, "tokens": 300, "spare": 16},
        # 63 samples of one long prompt, 32 layers of an 8B model.
        {"name": "fork_samples", "kind": "fork", "layers": 32, "heads": "8b", "page": 64, "slots": 64, "children": 63, "tokens": 4010, "spare": 70},
        # Two of four users leave, two others come.
        {"name": "turnover_small", "kind": "turnover", "page": 16, "slots": 4, "replaced": 2, "tokens": 200, "pages": 64},
        # A server's pool of a million tokens, a quarter of its 256 slots given to other users at once.
        {"name": "turnover_server", "kind": "turnover", "page": 16, "slots": 256, "replaced": 64, "tokens": 4000, "pages": 65536},
        # A few users left in a small pool: their pages move to its front.
        {"name": "compact_small", "kind": "compact", "layers": 2, "heads": "tiny", "page": 16, "pages": 96, "slots": 6, "tokens": 130},
        # An 8B model's pool, half in use after a busy hour, made dense so that its back half can be handed out.
        {"name": "compact_pool", "kind": "compact", "layers": 32, "heads": "8b", "page": 16, "pages": 700, "slots": 24, "tokens": 500},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention"] * 4 + ["append", "fork", "turnover", "compact"])
    page = rng.choice([16, 32, 64, 128])
    heads = rng.choice(sorted(HEADS))
    if kind == "attention":
        groups = _log(rng, 1, 8)
        case = {"kind": kind, "heads": heads, "page": page, "groups": groups, "per": _log(rng, 1, max(1, 128 // groups)),
                "shared": rng.choice([0, _log(rng, 1, 65536), _log(rng, 64, 65536)]), "own": _log(rng, 1, 2000)}
        case["new"] = min(case["own"], rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 400)]))
        most = [c for c in listed() if c["name"] == "attention_long"][0]
        while any(_work(case)[k] > _work(most)[k] for k in ("bytes", "flops")):
            case["shared"], case["own"], case["per"] = case["shared"] // 2, max(1, case["own"] // 2), max(1, case["per"] - 1)
            case["new"] = min(case["own"], case["new"])
        return case
    if kind == "append":
        new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 400)])
        return {"kind": kind, "heads": heads, "page": page, "seqs": _log(rng, 1, max(1, min(128, 6000 // new))), "before": _log(rng, 1, 300), "new": new}
    if kind == "fork":
        slots = _log(rng, 2, 64)
        return {"kind": kind, "layers": _log(rng, 1, 16), "heads": heads, "page": page, "slots": slots, "children": rng.randint(1, slots),
                "tokens": _log(rng, 1, 3000), "spare": slots + rng.randint(0, 20)}
    if kind == "turnover":
        slots, tokens = _log(rng, 2, 256), _log(rng, 1, 4000)
        need = slots * (-(-tokens // page) + 1)
        return {"kind": kind, "page": page, "slots": slots, "replaced": rng.randint(1, slots), "tokens": tokens, "pages": min(65536, need + _log(rng, 1, need))}
    slots, tokens = _log(rng, 1, 24), _log(rng, 1, 500)
    return {"kind": kind, "layers": _log(rng, 1, 16), "heads": heads, "page": page, "pages": slots * (-(-tokens // page) + 1) + _log(rng, 1, 300),
            "slots": slots, "tokens": tokens}


# ---------------------------------------------------------------------------------------------------------------- lengths of a case
def _spread(n, most, step=7919):
    """`n` uneven lengths in 1 .. `most`, the longest among them."""
    return [most if i == 0 else 1 + (i * step) % most for i in range(n)]


def _attention_lengths(c):
    """Per sequence: tokens held, of which the last `new` (fewer where it holds fewer of its own) are asked about."""
    own_len = _spread(c["groups"] * c["per"], c["own"])
    return [(c["shared"] + n, min(n, c["new"])) for n in own_len]


def _work(c):
    if c["kind"] == "attention":
        nh, nkv = HEADS[c["heads"]]
        common = c["shared"] // c["page"] * c["page"] if c["per"] > 1 else 0
        lens = _attention_lengths(c)
        keys = (c["groups"] * common if c["per"] > 1 else 0) + sum(n - common for n, _ in lens)
        pairs = sum(new * n - new * (new - 1) // 2 for n, new in lens)
        return {"bytes": keys * nkv * D * 4 + len(lens) * c["new"] * nh * D * 4, "flops": pairs * nh * D * 4}
    if c["kind"] == "append":
        nh, nkv = HEADS[c["heads"]]
        t = sum(_spread(c["seqs"], c["new"]))
        return {"bytes": t * (2 * nh + 4 * nkv) * D * 2, "flops": t * (nh + nkv) * D * 3}
    if c["kind"] == "fork":
        nkv = HEADS[c["heads"]][1]
        row = c["layers"] * 2 * nkv * D * 2
        src, dst = _parents(c)
        lens = _spread(c["slots"], c["tokens"])
        part = {s: lens[s] % c["page"] for s in src}
        pairs = [(s, d) for s, d in zip(src, dst) if s != d]
        moved = sum(part[s] for s, _ in pairs) + sum(part[s] for s in {s for s, _ in pairs})
        return {"bytes": moved * row + 8 * sum(-(-lens[s] // c["page"]) for s, _ in pairs) + 8 * len(pairs), "flops": 0}
    if c["kind"] == "turnover":
        n = sum(-(-t // c["page"]) for t in _spread(c["replaced"], c["tokens"])) + sum(-(-t // c["page"]) for t in _spread(c["slots"], c["tokens"], 104729)[:c["replaced"]])
        return {"bytes": 12 * n + 4 * c["replaced"] * c["tokens"], "flops": 0}
    nkv = HEADS[c["heads"]][1]
    held = _held(c)
    move = sum(1 for p in held if p >= len(held))
    return {"bytes": move * c["layers"] * 2 * nkv * c["page"] * D * 2 * 2 + 4 * (c["pages"] + len(held)), "flops": 0}


def work(case):
    return _work(case)


def _held(c):
    """The pages that a fragmented pool has in use."""
    return random.Random(c["pages"] * 31 + c["slots"]).sample(range(c["pages"]), sum(-(-t // c["page"]) for t in _spread(c["slots"], c["tokens"])))


def _parents(c):
    """Who goes on from whom: a few parents, which go on from themselves."""
    r = random.Random(c["slots"] * 1009 + c["children"])
    dst = sorted(r.sample(range(c["slots"]), c["children"]))
    few = [0] if c["children"] < c["slots"] else r.sample(range(c["slots"]), max(1, c["slots"] // 3))
    return [d if d in few else r.choice(few) for d in dst], dst


# ---------------------------------------------------------------------------------------------------------------- state
def _cache(layers, nkv, pages, page, table, lengths, refs, pool):
    if not own:
        return None
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from models.pages import PagedCache
    cache = PagedCache(layers, nkv, pages, page_size=page, max_seqs=table.shape[0], max_pages=table.shape[1], device="cuda")
    cache.table.copy_(table), cache.lengths.copy_(lengths), cache.refs.copy_(refs)
    if pool is not None:
        cache.pool.copy_(pool)
    return cache


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    half = dict(dtype=torch.float16, device="cuda", generator=gen)
    s = {"case": c}
    nh, nkv = HEADS[c.get("heads", "single")]
    page = c["page"]
    layers = c.get("layers", 1)
    if c["kind"] == "attention":
        n = c["groups"] * c["per"]
        lens = _attention_lengths(c)
        whole = c["shared"] // page
        pages = c["groups"] * whole + sum(-(-t // page) - whole for t, _ in lens) + 3
        width = max(-(-t // page) for t, _ in lens)
        free = list(range(pages))
        r.shuffle(free)                                        # (a pool that has been in use for a while)
        rows, refs = [], [0] * pages
        for g in range(c["groups"]):
            common = [free.pop() for _ in range(whole)]
            for t, _ in lens[g * c["per"]:(g + 1) * c["per"]]:
                row = common + [free.pop() for _ in range(-(-t // page) - whole)]
                for p in row:
                    refs[p] += 1
                rows.append(row + [-1] * (width - len(row)))
        s["positions"] = _ints([[t - new + j if j < new else -1 for j in range(c["new"])] for t, new in lens]).view(-1)
        s["q"] = torch.randn((n * c["new"], nh * D), **half) * 2
        s["slots"] = _ints(list(range(n)))
        s["starts"] = _ints([g * c["per"] for g in range(c["groups"] + 1)])
        s["shared"] = _ints([whole * page if c["per"] > 1 else 0] * c["groups"])
        lengths = [t for t, _ in lens]
    elif c["kind"] == "append":
        n = c["seqs"]
        new = _spread(n, c["new"])
        before = _spread(n, c["before"], 104729)
        need = [-(-(a + b) // page) for a, b in zip(before, new)]
        pages, width = sum(need) + 2, max(need)
        free = list(range(pages))
        r.shuffle(free)
        rows = [[free.pop() for _ in range(k)] + [-1] * (width - k) for k in need]
        refs = [0] * pages
        for row in rows:
            for p in row:
                if p >= 0:
                    refs[p] = 1
        s["positions"] = _ints([[b + j if j < k else -1 for j in range(c["new"])] for b, k in zip(before, new)]).view(-1)
        s["qkv"] = torch.randn((n * c["new"], (nh + 2 * nkv) * D), **half)
        s["inv_freq"] = (1.0 / (THETA ** (torch.arange(0, D, 2, dtype=torch.float32) / D))).cuda()
        s["slots"] = _ints(r.sample(range(n), n))
        by = s["slots"].tolist()                               # the i-th sequence of the batch lives in slot by[i]
        rows = [rows[by.index(k)] for k in range(n)]
        lengths = [(before[by.index(k)] + new[by.index(k)]) for k in range(n)]
    else:
        n = c["slots"]
        lens = _spread(n, c["tokens"], 104729 if c["kind"] == "turnover" else 7919)
        need = [-(-t // page) for t in lens]
        pages = c["pages"] if "pages" in c else sum(need) + c["spare"]
        width = max(max(need), -(-c["tokens"] // page)) + 1
        free = _held(c) if c["kind"] == "compact" else r.sample(range(pages), sum(need))
        rows = [[free.pop() for _ in range(k)] + [-1] * (width - k) for k in need]
        refs = [0] * pages
        for row in rows:
            for p in row:
                if p >= 0:
                    refs[p] = 1
        lengths = lens
        if c["kind"] == "fork":
            src, dst = _parents(c)
            s["src"], s["dst"] = _ints(src), _ints(dst)
        elif c["kind"] == "turnover":
            nkv = 1
            s["slots"] = _ints(list(range(c["replaced"])))
            s["tokens"] = _ints(_spread(c["replaced"], c["tokens"]))
    s["table"], s["lengths"], s["refs"] = _ints(rows), _ints(lengths), _ints(refs)
    s["pool"] = None
    if c["kind"] != "turnover":
        s["pool"] = torch.randn((layers, 2, pages, nkv, page, D), **half)
    s["cache"] = _cache(layers, nkv, pages, page, s["table"], s["lengths"], s["refs"], s["pool"])
    if own:
        s["pool"] = None
        if c["kind"] == "compact":
            s["book"] = s["cache"].book.clone()
    return s


# ---------------------------------------------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    c, cache = s["case"], s["cache"]
    if c["kind"] == "attention":
        return cache.attention(0, s["q"], s["positions"], s["slots"], group_starts=s["starts"], shared=s["shared"])
    if c["kind"] == "append":
        q = cache.rope_append(0, s["qkv"], s["positions"], s["inv_freq"], s["slots"])
        return q, cache.pool
    if c["kind"] == "fork":
        cache.fork(s["src"], s["dst"])
        return cache.table, cache.lengths, cache.refs, cache.pool
    if c["kind"] == "turnover":
        cache.free(s["slots"])
        positions = cache.reserve(s["slots"], s["tokens"], tokens_per_seq=c["tokens"])
        return cache.table, cache.lengths, cache.refs, positions
    cache.book.copy_(s["book"])                                # the fragmented pool once more; its pages still hold what they held
    cache.compact()
    return cache.table, cache.lengths, cache.refs, cache.pool


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _gather(s, which, slot, first, last):
    """K (0) or V (1) of the tokens first .. last - 1 of a slot, fp32 [KV heads, tokens, D]."""
    page = s["case"]["page"]
    p0, p1 = first // page, -(-last // page)
    t = s["pool"][0, which][s["table"][slot, p0:p1].long()].float()        # [pages, KV heads, page, D]
    t = t.permute(1, 0, 2, 3).reshape(t.shape[1], -1, D)
    return t[:, first - p0 * page:last - p0 * page]


def _attention_plain(s):
    c = s["case"]
    nh, nkv = HEADS[c["heads"]]
    R, per, new = nh // nkv, c["per"], c["new"]
    common = c["shared"] // c["page"] * c["page"] if per > 1 else 0
    lens = _attention_lengths(c)
    q = s["q"].float().view(-1, new, nkv, R, D).permute(0, 2, 1, 3, 4).reshape(-1, nkv, new * R, D) / math.sqrt(D)
    pos = s["positions"].view(-1, new, 1).expand(-1, new, R).reshape(-1, new * R, 1)
    out = torch.empty_like(q)
    for g in range(c["groups"]):
        at = slice(g * per, (g + 1) * per)
        if common:                                             # the shared pages, once for all rows of the group
            rows = q[at].transpose(0, 1).reshape(nkv, -1, D)
            sc = rows @ _gather(s, 0, g * per, 0, common).transpose(1, 2)
            top = sc.amax(-1, keepdim=True)
            w = torch.exp(sc - top)
            part = [x.view(nkv, per, new * R, -1).transpose(0, 1) for x in (top, w.sum(-1, keepdim=True), w @ _gather(s, 1, g * per, 0, common))]
        for i in range(at.start, at.stop):
            k, v = (_gather(s, h, i, common, lens[i][0]) for h in (0, 1))
            sc = q[i] @ k.transpose(1, 2)
            ahead = torch.arange(common, lens[i][0], device="cuda") > pos[i]
            sc = torch.where(ahead, torch.full_like(sc, float("-inf")), sc)
            top = sc.amax(-1, keepdim=True)
            if common:
                top = torch.maximum(top, part[0][i - at.start])
            w = torch.where(ahead, torch.zeros_like(sc), torch.exp(sc - top))
            num, den = w @ v, w.sum(-1, keepdim=True)
            if common:
                f = torch.exp(part[0][i - at.start] - top)
                num, den = num + f * part[2][i - at.start], den + f * part[1][i - at.start]
            out[i] = torch.where(pos[i] < 0, torch.zeros_like(num), num / den)
    return out.view(-1, nkv, new, R, D).permute(0, 2, 1, 3, 4).reshape(-1, nh * D).half()


def _append_plain(s):
    c = s["case"]
    nh, nkv = HEADS[c["heads"]]
    pos = s["positions"].long()
    x = s["qkv"].float().view(-1, nh + 2 * nkv, 2, D // 2)
    ang = pos.double()[:, None] * s["inv_freq"].double()       # (positions times frequencies lose their fraction in 32 bits)
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    a, b = x[:, :nh + nkv, 0], x[:, :nh + nkv, 1]
    rot = torch.stack((a * cos - b * sin, b * cos + a * sin), 2).view(-1, nh + nkv, D).half()
    on = (pos >= 0).nonzero().view(-1)
    slot = s["slots"].long().repeat_interleave(c["new"])[on]
    page = s["table"][slot, pos[on] // c["page"]].long()
    s["pool"][0, 0, page, :, pos[on] % c["page"]] = rot[on, nh:]
    s["pool"][0, 1, page, :, pos[on] % c["page"]] = s["qkv"].view(-1, nh + 2 * nkv, D)[on, nh + nkv:]
    q = torch.where((pos >= 0)[:, None, None], rot[:, :nh], torch.zeros_like(rot[:, :nh]))
    return q.reshape(-1, nh * D), s["pool"]


def _count(pages, rows):
    return torch.bincount(rows[rows >= 0].long(), minlength=pages).int()


def _fork_plain(s):
    c, table, lengths, refs = s["case"], s["table"], s["lengths"], s["refs"]
    page = c["page"]
    on = (s["src"] != s["dst"]).nonzero().view(-1)
    src, dst = s["src"][on].long(), s["dst"][on].long()
    rows, length = table[src], lengths[src]
    k = torch.arange(table.shape[1], device="cuda")
    full, part = (length // page)[:, None], length % page
    keep = torch.where(k < full, rows, torch.full_like(rows, -1))
    refs += _count(refs.numel(), keep) - _count(refs.numel(), table[dst])
    with_part = (part > 0).nonzero().view(-1)
    last = rows.gather(1, full.long().clamp(max=rows.shape[1] - 1))[with_part, 0].long()
    read = torch.zeros_like(refs).index_fill_(0, last, 1)
    new = ((refs == 0) & (read == 0)).nonzero().view(-1)[:with_part.numel()]
    refs[new] = 1
    keep[with_part, full[with_part, 0].long()] = new.int()
    table[dst], lengths[dst] = keep, length
    filled = torch.arange(page, device="cuda") < part[with_part][:, None]  # [children, rows]
    for i in range(new.numel()):
        s["pool"][:, :, new[i], :, filled[i]] = s["pool"][:, :, last[i], :, filled[i]]
    return table, lengths, refs, s["pool"]


def _turnover_plain(s):
    c, table, lengths, refs, slots = s["case"], s["table"], s["lengths"], s["refs"], s["slots"].long()
    refs -= _count(refs.numel(), table[slots])
    table[slots], lengths[slots] = -1, 0
    need = (s["tokens"] + c["page"] - 1) // c["page"]
    k = torch.arange(table.shape[1], device="cuda")
    take = k < need[:, None]
    new = (refs == 0).nonzero().view(-1)[:int(need.sum())]
    refs[new] = 1
    rows = table[slots]
    rows[take] = new.int()
    table[slots], lengths[slots] = rows, s["tokens"]
    j = torch.arange(c["tokens"], device="cuda", dtype=torch.int32)
    return table, lengths, refs, torch.where(j < s["tokens"][:, None], j, torch.full_like(j, -1)).view(-1)


def _compact_plain(s):
    table, refs = s["table"].clone(), s["refs"].clone()
    used = refs > 0
    n = int(used.sum())
    at = torch.arange(refs.numel(), device="cuda")
    src, dst = at[used & (at >= n)], at[~used & (at < n)]
    s["pool"][:, :, dst] = s["pool"][:, :, src]
    refs[dst], refs[src] = refs[src], 0
    where = at.int().clone()
    where[src] = dst.int()
    table = torch.where(table >= 0, where[table.clamp(min=0).long()], table)
    return table, s["lengths"], refs, s["pool"]


def run(state):
    if own:
        return _run_own(state)
    return {"attention": _attention_plain, "append": _append_plain, "fork": _fork_plain, "turnover": _turnover_plain,
            "compact": _compact_plain}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------------------- from the definition
def _state(case, seed):
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def _exact_attention(s):
    c = s["case"]
    nh, nkv = HEADS[c["heads"]]
    pool = s["pool"][0]
    out = torch.zeros((s["positions"].numel(), nh, D), dtype=torch.float64, device="cuda")
    positions, table = s["positions"].tolist(), s["table"].tolist()
    for i in range(len(table)):
        t = [(i * c["new"] + j, positions[i * c["new"] + j]) for j in range(c["new"]) if positions[i * c["new"] + j] >= 0]
        keys = t[-1][1] + 1
        pages = torch.tensor(table[i][:-(-keys // c["page"])], device="cuda")
        limit = torch.tensor([p for _, p in t], device="cuda")[None, :, None]
        for h in range(nkv):
            k, v = (pool[w, pages, h].reshape(-1, D)[:keys].double() for w in (0, 1))
            q = s["q"].view(-1, nh, D)[[r for r, _ in t], h * (nh // nkv):(h + 1) * (nh // nkv)].double().transpose(0, 1)
            sc = torch.einsum("rtd,kd->rtk", q, k) / math.sqrt(D)
            sc.masked_fill_(torch.arange(keys, device="cuda") > limit, float("-inf"))
            o = torch.einsum("rtk,kd->trd", torch.softmax(sc, -1), v)
            out[[r for r, _ in t], h * (nh // nkv):(h + 1) * (nh // nkv)] = o
    return out.view(-1, nh * D)


def _exact_append(s):
    c = s["case"]
    nh, nkv = HEADS[c["heads"]]
    pool = s["pool"].double()
    x = s["qkv"].double().view(-1, nh + 2 * nkv, D)
    q = torch.zeros((x.shape[0], nh, D), dtype=torch.float64, device="cuda")
    freq = s["inv_freq"].double().tolist()
    slots, table = s["slots"].tolist(), s["table"].tolist()
    where = s["positions"].tolist()
    turn = torch.zeros((x.shape[0], D // 2), dtype=torch.complex128)
    for t, p in enumerate(where):
        turn[t] = torch.tensor([complex(math.cos(p * f), math.sin(p * f)) for f in freq], dtype=torch.complex128)
    z = torch.complex(x[:, :nh + nkv, :D // 2], x[:, :nh + nkv, D // 2:]) * turn.cuda()[:, None]
    z = torch.cat((z.real, z.imag), -1)
    for t, p in enumerate(where):
        if p >= 0:
            at = table[slots[t // c["new"]]][p // c["page"]]
            q[t] = z[t, :nh]
            pool[0, 0, at, :, p % c["page"]], pool[0, 1, at, :, p % c["page"]] = z[t, nh:], x[t, nh + nkv:]
    return q.view(-1, nh * D), pool


def _exact_pages(s):
    """The bookkeeping one page at a time; what lands where is moved in a copy of the pool."""
    c, page = s["case"], s["case"]["page"]
    table, lengths, refs = s["table"].tolist(), s["lengths"].tolist(), s["refs"].tolist()
    pool = s["pool"].double() if s["pool"] is not None else None
    width = len(table[0])
    move = []                                                  # (from, to, rows)
    extra = None

    def drop(slot):
        for p in table[slot]:
            if p >= 0:
                refs[p] -= 1
        table[slot], lengths[slot] = [-1] * width, 0

    if c["kind"] == "fork":
        old, old_len = [list(r) for r in table], list(lengths)
        pairs = [(a, b) for a, b in zip(s["src"].tolist(), s["dst"].tolist()) if a != b]
        for _, b in pairs:
            drop(b)
        for a, b in pairs:
            for i in range(old_len[a] // page):
                table[b][i] = old[a][i]
                refs[old[a][i]] += 1
            lengths[b] = old_len[a]
        read = {old[a][old_len[a] // page] for a, _ in pairs if old_len[a] % page}
        free = (p for p in range(len(refs)) if refs[p] == 0 and p not in read)
        for a, b in pairs:
            if old_len[a] % page:
                p = next(free)
                move.append((old[a][old_len[a] // page], p, old_len[a] % page))
                table[b][old_len[a] // page] = p
        for _, p, _ in move:
            refs[p] = 1
    elif c["kind"] == "turnover":
        for slot in s["slots"].tolist():
            drop(slot)
        free = iter([p for p in range(len(refs)) if refs[p] == 0])
        extra = []
        for slot, t in zip(s["slots"].tolist(), s["tokens"].tolist()):
            for i in range(-(-t // page)):
                table[slot][i] = next(free)
                refs[table[slot][i]] = 1
            lengths[slot] = t
            extra += [j if j < t else -1 for j in range(c["tokens"])]
    else:
        n = sum(1 for x in refs if x > 0)
        pairs = list(zip([p for p in range(n, len(refs)) if refs[p] > 0], [p for p in range(n) if refs[p] == 0]))
        to = dict(pairs)
        table = [[to.get(p, p) for p in row] for row in table]
        for a, b in pairs:
            refs[b], refs[a] = refs[a], 0
            move.append((a, b, page))
    if pool is not None:
        was = pool.clone() if c["kind"] == "fork" else pool
        for a, b, rows in move:
            pool[:, :, b, :, :rows] = was[:, :, a, :, :rows]
    i32 = dict(dtype=torch.int32)
    return torch.tensor(table, **i32), torch.tensor(lengths, **i32), torch.tensor(refs, **i32), torch.tensor(extra, **i32) if extra is not None else pool


def exact(case, seed):
    s = _state(case, seed)
    return {"attention": _exact_attention, "append": _exact_append}.get(case["kind"], _exact_pages)(s)
