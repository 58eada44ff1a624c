"""The paged KV cache (models/pages.py; csrc/pages.cu, csrc/attention_pages.cu) against restatements in plain Python and 64 bits.

Bounds, counted in half steps of fp16 (2^-11 of a value, 2^-25 below 2^-14):
  rotary embedding   one rounding of a value computed in fp32: 2^-11 |x| + 2^-25, and 2^-21 of the pair's length for cos, sin and the sum (angles to
                     2^-25 of half a turn and two ulp of sincosf, 4e-7 together)
  attention          weights rounded to fp16 (2^-11 of each: 2^-11 of the sum of weights times |v|), the result rounded once (2^-11 of it); scores and sums in
                     fp32 add less than 2^-16 of that sum for scores below 2^6; weights that fp16 cannot hold are below 2^-35 of the largest
"""
import random

import pytest
import torch

from tests.pages_model import D, Model, attention, rope

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -11


def make(layers=1, n_kv=2, pages=40, page=16, max_seqs=6, max_pages=12, seed=1):
    from models.pages import PagedCache
    c = PagedCache(layers, n_kv, pages, page_size=page, max_seqs=max_seqs, max_pages=max_pages)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.pool.copy_(torch.randn(c.pool.shape, device="cuda", generator=g).half())
    return c, Model(pages, page, max_seqs, max_pages, c.pool.cpu().clone())


def same(c, m):
    assert c.lengths.tolist() == m.lengths
    assert c.refs.tolist() == m.refs
    assert c.table.tolist() == m.table
    assert torch.equal(c.pool.cpu(), m.pool)
    assert int(c.status) == m.status


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ bookkeeping
def test_reserve_in_order_and_positions():
    c, m = make()
    assert c.reserve([3, 1], ints([17, 33]), tokens_per_seq=20).tolist() == m.reserve([3, 1], [17, 33], 20)
    same(c, m)
    assert c.reserve([1, 0, 3], 15, tokens_per_seq=3).tolist() == m.reserve([1, 0, 3], [15] * 3, 3)
    same(c, m)
    assert c.reserve([0], 0) is None
    assert c.reserve(None, 1, tokens_per_seq=1).tolist() == m.reserve(list(range(6)), [1] * 6, 1)
    same(c, m)


def test_calls_that_cannot_be_done_change_nothing():
    c, m = make(pages=10)
    c.reserve([0, 1], ints([70, 50])), m.reserve([0, 1], [70, 50], 0)
    same(c, m)
    assert c.reserve([2], 17, tokens_per_seq=2).tolist() == [-1, -1]          # one page is left
    m.status |= 1
    same(c, m)
    with pytest.raises(RuntimeError, match="fewer free pages"):
        c.check()
    c.check()
    m.status = 0
    for call in (lambda: c.reserve([3], 193), lambda: c.reserve([0], 123)):
        call()
        with pytest.raises(RuntimeError, match="beyond 12 pages"):
            c.check()
    for call in (lambda: c.free(ints([0, 0])), lambda: c.free(ints([6])), lambda: c.reserve(ints([1, -1]), 1), lambda: c.reserve(ints([0, 1]), ints([3, -1])),
                 lambda: c.fork(ints([0, 1]), ints([2, 2])), lambda: c.fork(ints([6]), ints([2])), lambda: c.copy(ints([0]), ints([-1]))):
        call()
        with pytest.raises(RuntimeError, match="slot"):
            c.check()
        same(c, m)
    for call in (lambda: c.copy([0], [2]), lambda: c.fork([0, 0], [2, 3])):      # five pages, and two part-filled ones
        call()
        with pytest.raises(RuntimeError, match="fewer free pages"):
            c.check()
        same(c, m)
    c.fork([0], [1])                                           # the child's own pages come back first: there is room
    m.fork([0], [1])
    same(c, m)


@pytest.mark.parametrize("share", [True, False])
def test_fork_all_at_once(share):
    """Children that are parents of others (a swap, a chain), that stay what they are, that hold their parent's pages already, and an empty parent."""
    c, m = make(layers=2, pages=90, max_seqs=8)
    c.reserve([0, 1, 2, 3], ints([40, 70, 16, 5])), m.reserve([0, 1, 2, 3], [40, 70, 16, 5], 0)
    for src, dst in (([0, 1, 1, 0], [1, 0, 4, 5]), ([0, 1, 2, 4], [0, 2, 3, 1]), ([5, 5, 5], [0, 1, 2]), ([7, 3], [3, 6]), ([3], [3])):
        (c.fork if share else c.copy)(src, dst)
        m.fork(src, dst, share)
        same(c, m)


@pytest.mark.parametrize("page,pages,seqs,width,seed", [(16, 50, 5, 9, 0), (32, 30, 9, 6, 1), (128, 12, 4, 3, 2), (16, 40000, 40, 300, 3), (256, 9, 3, 4, 4)])
def test_any_order_of_calls(page, pages, seqs, width, seed):
    r = random.Random(seed)
    c, m = make(1, 1, pages, page, seqs, width, seed) if pages < 1000 else make(1, 1, pages, page, seqs, width, seed)
    for step in range(30):
        k = r.randint(1, seqs)
        some = r.sample(range(seqs), k)
        what = r.choice(["reserve", "reserve", "reserve", "free", "fork", "fork", "copy", "compact"])
        if what == "reserve":
            t = [r.choice([0, 1, r.randint(0, page), r.randint(0, width * page // 2)]) for _ in some]
            tps = r.choice([1, 7])
            assert c.reserve(ints(some), ints(t), tokens_per_seq=tps).tolist() == m.reserve(some, t, tps)
        elif what == "free":
            some = some[:max(1, k // 3)]
            c.free(ints(some)), m.free(some)
        elif what == "compact":
            c.compact(), m.compact()
        else:
            src = [r.randrange(seqs) for _ in some]
            getattr(c, what)(ints(src), ints(some)), m.fork(src, some, what == "fork")
        if pages < 1000 or step % 10 == 9:
            same(c, m)
    starts, slots = [0, 2, 2 + seqs // 2, seqs], r.sample(range(seqs), seqs)
    starts = sorted(min(s, seqs) for s in starts)
    got = c.common(ints(slots), ints(starts)).tolist()
    assert got == [m.common(slots[a:b]) for a, b in zip(starts, starts[1:])]


def test_common_pages():
    c, m = make(pages=60, max_seqs=8)
    c.reserve([0], 70), m.reserve([0], [70], 0)
    c.fork([0, 0, 0], [1, 2, 5])
    c.reserve([0, 1, 2, 5, 6], 30)
    c.fork([2], [3])
    assert c.common([0, 1, 2, 3, 5, 6, 6], ints([0, 2, 4, 5, 7])).tolist() == [64, 96, 0, 16]
    assert c.common([0, 6, 2], ints([0, 3])).tolist() == [0]
    assert c.common([2, 3, 2], ints([0, 3])).tolist() == [96]
    c.check()


def test_bookkeeping_replayed():
    """Captured once, replayed: what a call does follows the state at that time."""
    c, m = make(pages=60)
    slots = ints([0, 1, 2, 3])
    c.reserve(slots, 14), m.reserve([0, 1, 2, 3], [14] * 4, 0)
    g = torch.cuda.CUDAGraph()
    src, dst, gone = ints([0, 0, 1]), ints([2, 3, 4]), ints([5])
    with torch.cuda.graph(g):
        pos = c.reserve(slots, 3, tokens_per_seq=1)
        c.fork(src, dst)
        c.free(gone)
        c.compact()
    for _ in range(9):
        g.replay()
        want = m.reserve([0, 1, 2, 3], [3] * 4, 1)
        m.fork([0, 0, 1], [2, 3, 4]), m.free([5]), m.compact()
        assert pos.tolist() == want
        same(c, m)


# ------------------------------------------------------------------ rotary embedding and append
@pytest.mark.parametrize("B,tps,nh,nkv,page,far", [(3, 1, 4, 2, 16, 0), (2, 37, 6, 3, 32, 0), (1, 5, 64, 8, 128, 0), (5, 4, 15, 3, 16, 150), (2, 3, 1, 1, 256, 70000)])
def test_rope_append(B, tps, nh, nkv, page, far):
    width = -(-(far + tps + 60) // page)
    c, m = make(2, nkv, B * width + 1, page, B + 2, width, seed=B + tps)
    r = random.Random(tps)
    slots = r.sample(range(B + 2), B)
    new = [r.randint(0, tps) if b else tps for b in range(B)]
    c.reserve(slots, far + 3)
    pos = c.reserve(slots, ints(new), tokens_per_seq=tps)
    g = torch.Generator(device="cuda").manual_seed(7)
    qkv = torch.randn((B * tps, (nh + 2 * nkv) * D), device="cuda", generator=g).half()
    inv = 500000.0 ** (-torch.arange(0, D, 2, device="cuda").float() / D)
    pool, kept = c.pool.clone(), qkv.clone()
    q = c.rope_append(1, qkv, pos, inv, slots, scaling=1.0)
    c.check()
    x = qkv.view(B * tps, nh + 2 * nkv, D)
    rot = rope(x[:, :nh + nkv], pos, inv)
    size = (x[:, :nh + nkv].double().view(B * tps, nh + nkv, 2, D // 2) ** 2).sum(2, keepdim=True).sqrt().expand(-1, -1, 2, -1).reshape(rot.shape)
    bound = HALF * rot.abs() + 2.0 ** -25 + 2.0 ** -21 * size
    want = pool.double()
    lim = torch.zeros_like(want)
    for t, p in enumerate(pos.tolist()):
        if p < 0:
            assert not q[t].any()
            rot[t], bound[t] = 0, 0
            continue
        at = c.table[slots[t // tps], p // page]
        want[1, 0, at, :, p % page], lim[1, 0, at, :, p % page] = rot[t, nh:], bound[t, nh:]
        want[1, 1, at, :, p % page] = x[t, nh + nkv:].double()
    assert ((q.view(B * tps, nh, D).double() - rot[:, :nh]).abs() <= bound[:, :nh]).all()
    assert ((c.pool.double() - want).abs() <= lim).all()      # (every other place: as it was)
    assert torch.equal(qkv, kept)


def test_rope_append_keeps_to_the_table():
    """A position without a page is not stored, and said."""
    c, m = make(pages=8)
    c.reserve([0], 20)
    inv = 500000.0 ** (-torch.arange(0, D, 2, device="cuda").float() / D)
    qkv = torch.randn((3, 6 * D), device="cuda").half()
    pool = c.pool.clone()
    q = c.rope_append(0, qkv, ints([32, 5000, 3]), inv, ints([0, 0, 1]))
    assert torch.equal(c.pool, pool) and q.any(1).all()
    with pytest.raises(RuntimeError, match="no page"):
        c.check()
    c.rope_append(0, qkv[:1], ints([0]), inv, ints([99]))
    assert torch.equal(c.pool, pool)
    with pytest.raises(RuntimeError, match="no page"):
        c.check()


# ------------------------------------------------------------------ attention
def batch(groups, per, shared, own, tps, nh, nkv, page, seed=0, layers=1, spare=3):
    """Groups of sequences that fork from a common text, go on for 1 .. `own` tokens and ask about their last ones (at most `tps`)."""
    from models.pages import PagedCache
    r = random.Random(seed)
    n = groups * per
    lens = [own if i == 0 else r.randint(1, own) for i in range(n)]
    width = -(-(shared + own) // page)
    c = PagedCache(layers, nkv, groups * (-(-shared // page)) + n * (-(-own // page) + 1) + spare, page_size=page, max_seqs=n + 1, max_pages=width)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    c.pool.copy_(torch.randn(c.pool.shape, device="cuda", generator=g).half())
    slots = r.sample(range(n + 1), n)
    for k in range(groups):
        mine = slots[k * per:(k + 1) * per]
        if shared:
            c.reserve(mine[:1], shared)
            if per > 1:
                c.fork(mine[:1] * (per - 1), mine[1:])
        c.reserve(mine, ints(lens[k * per:(k + 1) * per]))
    c.check()
    # pages of no sequence, and tokens behind a sequence's last: never read
    c.pool[:, :, (c.refs == 0).nonzero().view(-1)] = float("nan")
    total = [shared + x for x in lens]
    for i, s in enumerate(slots):
        if total[i] % page:
            c.pool[:, :, c.table[s, total[i] // page].long(), :, total[i] % page:] = float("nan")
    pos = ints([[total[i] - min(tps, lens[i]) + j if j < min(tps, lens[i]) else -1 for j in range(tps)] for i in range(n)]).view(-1)
    q = torch.randn((n * tps, nh * D), device="cuda", generator=g).half() * 2
    starts = ints([k * per for k in range(groups + 1)])
    return c, q, pos, slots, starts


def close(out, ref, keys):
    o, mag = ref
    err = (out.double() - o).abs()
    bound = (HALF + 2.0 ** -16) * (mag + o.abs()) + 2.0 ** -25 + keys * 2.0 ** -33
    assert torch.isfinite(out).all()
    worst = (err / bound).max().item()
    assert worst <= 1.0, worst


CASES = [
    # groups, per, shared, own, tps, nh, nkv, page
    (1, 1, 0, 1, 1, 1, 1, 16), (1, 3, 0, 17, 1, 4, 2, 16), (1, 4, 256, 40, 1, 4, 2, 16), (2, 5, 100, 70, 1, 32, 8, 32),
    (1, 2, 1000, 1, 1, 8, 8, 64), (3, 7, 300, 130, 1, 15, 3, 64), (1, 40, 2000, 300, 1, 32, 8, 64), (1, 70, 700, 90, 1, 64, 8, 128),
    (2, 3, 513, 50, 3, 8, 1, 256), (1, 6, 130, 33, 7, 32, 8, 16), (4, 1, 900, 40, 1, 16, 8, 32), (1, 9, 64, 20, 15, 8, 2, 64),
    (1, 2, 5, 3, 1, 4, 2, 16), (2, 2, 16, 16, 1, 4, 2, 16), (6, 2, 48, 5, 2, 21, 3, 16),
    (1, 1, 20000, 9, 1, 8, 2, 64), (1, 33, 9000, 9, 1, 8, 1, 128),
    # many rows per sequence
    (1, 3, 100, 90, 64, 4, 4, 16), (1, 2, 777, 300, 300, 32, 8, 32), (2, 3, 40, 200, 130, 15, 3, 64), (1, 1, 3001, 65, 65, 8, 8, 128), (5, 1, 0, 129, 129, 8, 1, 16),
    (1, 8, 4001, 300, 300, 32, 8, 32),
]


@pytest.mark.parametrize("case", CASES)
def test_attention(case):
    groups, per, shared, own, tps, nh, nkv, page = case
    c, q, pos, slots, starts = batch(*case, seed=len(CASES) + CASES.index(case))
    common = c.common(slots, starts)
    assert common.tolist() == [shared // page * page if per > 1 else 0] * groups
    ref = attention(c, 0, q, pos, slots, nh)
    close(c.attention(0, q, pos, slots, group_starts=starts, shared=common), ref, shared + own)
    out = torch.full((q.shape[0] + 2, nh * D), 7.0, dtype=torch.float16, device="cuda")
    close(c.attention(0, q, pos, ints(slots), out=out[1:-1]), ref, shared + own)        # nothing said of what is shared
    assert (out[0] == 7.0).all() and (out[-1] == 7.0).all()
    empty = pos < 0
    assert not out[1:-1][empty].any()
    c.check()
