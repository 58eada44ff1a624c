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


@pytest.mark.parametrize("case", [(1, 3, 90, 70, 64, 8, 4, 32), (1, 5, 300, 40, 40, 8, 2, 16), (1, 4, 200, 30, 6, 8, 2, 16), (2, 9, 640, 20, 1, 8, 2, 128)])
def test_what_lies_behind_a_sequence_does_not_matter(case):
    """Finite leftovers, infinities and NaN behind the last token and in free pages: the same bits."""
    outs = []
    for fill in (0.0, 60000.0, float("inf"), float("nan")):
        c, q, pos, slots, starts = batch(*case, seed=77)
        c.pool[torch.isnan(c.pool)] = fill
        outs.append(c.attention(0, q, pos, slots, group_starts=starts, shared=c.common(slots, starts)))
    assert torch.isfinite(outs[0]).all() and all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("tps,groups", [(6, True), (6, False), (60, False), (1, True), (5, True)])
def test_values_that_are_not_finite_reach_the_tokens_that_see_them(tps, groups):
    c, q, pos, slots, starts = batch(1, 4, 256, 60, tps, 8, 2, 32, seed=5)
    common = c.common(slots, starts)
    say = dict(group_starts=starts, shared=common) if groups else {}
    o, mag = attention(c, 0, q, pos, slots, 8)                 # (dims do not mix: those that stay finite stay what they are)
    at = int(pos.view(4, tps)[0, tps // 2])                    # the first sequence's own, seen from the middle token on
    page = int(c.table[slots[0], at // 32])
    c.pool[0, 1, page, 1, at % 32, 3] = float("inf")
    c.pool[0, 1, int(c.table[slots[0], 2]), 0, 5, 7] = float("-inf")           # a shared one, seen by all
    got = c.attention(0, q, pos, slots, **say).view(4, tps, 2, 4, D)
    bad = ~torch.isfinite(got)
    expect = torch.zeros_like(bad)
    expect[0, tps // 2:, 1, :, 3] = True
    expect[..., 0, :, 7] = True
    expect[pos.view(4, tps) < 0] = False
    assert torch.equal(bad, expect)
    bad = bad.view(4 * tps, -1)
    close(got.view(4 * tps, -1).masked_fill(bad, 0), (o.masked_fill(bad, 0), mag), 316)


@pytest.mark.parametrize("step", [0.02, 0.7, 9.0])
@pytest.mark.parametrize("tps", [1, 40])
def test_growing_scores(step, tps):
    """Scores that grow along the keys, slowly and fast: the reference of the weights lags behind and is moved in steps."""
    c, q, pos, slots, starts = batch(1, 5, 640, 90, tps, 8, 2, 64, seed=9)
    n = 730
    q *= 0.1
    q.view(-1, 8, D)[:, :, 0] = 8.0
    ramp = (torch.arange(n, device="cuda") * step * D ** 0.5 / 8.0).clamp(max=30000.0).half()
    for s in slots:
        for k in range(-(-n // 64)):
            p = int(c.table[s, k])
            if p >= 0:
                c.pool[0, 0, p, :, :, 0] = ramp[k * 64:(k + 1) * 64].new_zeros(64).copy_(torch.nn.functional.pad(ramp[k * 64:(k + 1) * 64], (0, max(0, (k + 1) * 64 - n))))
    common = c.common(slots, starts)
    o, mag = attention(c, 0, q, pos, slots, 8)
    out = c.attention(0, q, pos, slots, group_starts=starts, shared=common)
    # fp32 scores of up to 9 * 730 * log2(e): half a step of 2^-11 of them at most, in the exponent; eight products' and sums' worth
    slack = 1.0 + 8 * 2.0 ** -24 * (n * step * 1.4427) * 2.0 ** 11
    err = (out.double() - o).abs()
    assert (err <= slack * HALF * (mag + o.abs()) + 2.0 ** -24).all(), (err / (mag + o.abs() + 1e-9)).max()


def test_rows_apart_and_scales():
    c, q, pos, slots, starts = batch(1, 6, 300, 40, 2, 8, 2, 32, seed=11)
    common = c.common(slots, starts)
    wide = torch.full((q.shape[0], q.shape[1] + 3 * 8), 9.0, dtype=torch.float16, device="cuda")
    wide[:, 8:8 + q.shape[1]] = q
    view = wide[:, 8:8 + q.shape[1]]
    assert torch.equal(c.attention(0, q, pos, slots, group_starts=starts, shared=common), c.attention(0, view, pos, slots, group_starts=starts, shared=common))
    for scale in (0.01, 1.0):
        close(c.attention(0, q, pos, slots, scale=scale, group_starts=starts, shared=common), attention(c, 0, q, pos, slots, 8, scale), 340 if scale < 1 else 3400)


def test_any_batch_order_and_groups():
    """Groups of one, groups that share nothing, sequences in no group, a slot twice in a batch."""
    c, q, pos, slots, starts = batch(3, 4, 200, 50, 1, 8, 2, 16, seed=13)
    ref = attention(c, 0, q, pos, slots, 8)
    for cuts in ([0, 4, 8, 12], [0, 1, 4, 12], [2, 4], [0, 2, 8], [5, 5, 8, 8, 12]):
        g = ints(cuts)
        close(c.attention(0, q, pos, slots, group_starts=g, shared=c.common(slots, g)), ref, 250)
    twice = [slots[0], slots[0], slots[5], slots[0]]
    rows = [0, 0, 5, 0]
    out = c.attention(0, q[rows].contiguous(), pos[rows].contiguous(), ints(twice), group_starts=ints([0, 2, 4]), shared=c.common(ints(twice), ints([0, 2, 4])))
    close(out, (ref[0][rows], ref[1][rows]), 250)
    assert torch.equal(out[0], out[1])


def test_many_groups():
    c, q, pos, slots, starts = batch(70, 2, 40, 6, 1, 4, 2, 16, seed=15)
    close(c.attention(0, q, pos, slots, group_starts=starts, shared=c.common(slots, starts)), attention(c, 0, q, pos, slots, 4), 46)


def test_a_far_layer():
    """Elements of a pool beyond 2^31."""
    c, q, pos, slots, starts = batch(1, 3, 500, 60, 1, 8, 8, 256, seed=17, layers=2, spare=5000)
    assert c.pool[1].storage_offset() + c.pool[1].numel() > 2 ** 31
    c.pool[1, :, c.refs > 0] = c.pool[0, :, c.refs > 0]
    a, b = (c.attention(layer, q, pos, slots, group_starts=starts, shared=c.common(slots, starts)) for layer in (0, 1))
    assert torch.equal(a, b)
    close(b, attention(c, 1, q, pos, slots, 8), 560)


def test_replayed_and_on_other_streams():
    """Two graphs of the same cache replayed one after the other, and a call on a stream of its own: the same bits as the eager call."""
    c, q, pos, slots, starts = batch(2, 20, 700, 90, 1, 32, 8, 64, seed=19)
    sl, common = ints(slots), c.common(slots, starts)
    want = c.attention(0, q, pos, sl, group_starts=starts, shared=common)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c.attention(0, q, pos, sl, group_starts=starts, shared=common)
        graphs.append((g, out))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = c.attention(0, q, pos, sl, group_starts=starts, shared=common)
    for _ in range(3):
        for g, out in graphs:
            out.zero_()
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(other, want) and all(torch.equal(out, want) for _, out in graphs)


def test_two_calls_at_once():
    """Two streams, two batches, one cache that neither changes: every call has scratch of its own."""
    c, q, pos, slots, starts = batch(2, 20, 3000, 90, 1, 32, 8, 64, seed=21)
    sl, common = ints(slots), c.common(slots, starts)
    q2 = q.flip(0).contiguous()
    want = [c.attention(0, x, pos, sl, group_starts=starts, shared=common) for x in (q, q2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(c.attention(0, (q, q2)[k], pos, sl, group_starts=starts, shared=common))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[k]) for k in range(2) for o in got[k])


@pytest.mark.parametrize("case", [(1, 40, 700, 20, 1, 32, 8, 64), (1, 5, 200, 20, 1, 8, 2, 16), (1, 2, 200, 150, 100, 8, 2, 32), (1, 4, 300, 40, 6, 8, 2, 16)])
@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_entries_that_name_no_page(case, entry):
    """Read as keys and values of zeros, and said; what does not read them is what it was."""
    c, q, pos, slots, starts = batch(*case, seed=41)
    groups, per, shared, own, tps, nh, nkv, page = case
    common = c.common(slots, starts)
    c.check()
    last = slots[per - 1]
    k = int(c.lengths[last] - 1) // page
    kept = c.table.clone()
    c.table[last, k] = entry                                   # a page of the last sequence's own
    c.table[slots[0], 1] = entry                               # one that is shared, by its first sequence's row
    out = c.attention(0, q, pos, ints(slots), group_starts=starts, shared=common)
    with pytest.raises(RuntimeError, match="no page"):
        c.check()
    c.table.copy_(kept)
    free = int((c.refs == 0).nonzero()[0])
    c.pool[:, :, free] = 0
    c.table[last, k] = free
    for s in (slots if tps * (nh // nkv) < 64 and _shares(c, case) else slots[:1]):
        c.table[s, 1] = free
    close(out, attention(c, 0, q, pos, slots, nh), shared + own)


def _shares(c, case):
    """Whether a call reads the first sequence's pages for all of them: where that can save 2 MB (csrc/attention_pages.cu)."""
    groups, per, shared, own, tps, nh, nkv, page = case
    return (per - 1) * groups * c.max_pages * page * nkv * 512 > 2 << 20


@pytest.fixture(scope="module")
def impatient(tmp_path_factory):
    """The kernels with a wait that runs out (tests/native/pages_timeout.cu)."""
    import ctypes
    import os
    import shutil
    import subprocess
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not available")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    so = str(tmp_path_factory.mktemp("native") / "pages_timeout.so")
    subprocess.check_call([nvcc, "-std=c++17", "-O3", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC",
                           "-I", os.path.join(root, "include"), "-I", os.path.join(root, "sbvr-cpu-arm_b200", "csrc"),
                           "-o", so, os.path.join(root, "tests", "native", "pages_timeout.cu")])
    from sbvr import _lib
    lib = ctypes.CDLL(so)
    lib.sbvr_pages_attention_f16.argtypes = _lib.lib.sbvr_pages_attention_f16.argtypes
    return lib


# warps and barriers by their numbers: 128 rows: 0-3 weights, 4 MMAs, 5 K, 6 V; [2] K, V there, [2] K, V read, [2] scores, weights, outputs there, -, V to be
# looked through, queries.  256 rows: 0-7, 8, 9, 10; [5] each of the first four, [4] of the next three.
PROMPT, SHARED = (2, 2, 200, 150, 100, 8, 2, 32), (1, 40, 3000, 20, 1, 32, 8, 64)


@pytest.mark.parametrize("case,warp,bar,parity", [
    (PROMPT, 4, 0, 0), (PROMPT, 4, 3, 0), (PROMPT, 4, 10, 0), (PROMPT, 4, 16, 0), (PROMPT, 5, 4, 0), (PROMPT, 6, 7, 0), (PROMPT, 6, 15, 0), (PROMPT, 0, 8, 1),
    (PROMPT, 3, 9, 0), (PROMPT, 2, 12, 0),
    (SHARED, 8, 1, 0), (SHARED, 8, 7, 0), (SHARED, 8, 26, 0), (SHARED, 8, 35, 0), (SHARED, 9, 10, 0), (SHARED, 10, 16, 0), (SHARED, 1, 20, 0), (SHARED, 6, 23, 1),
    (SHARED, 4, 30, 0)])
def test_a_wait_that_runs_out_costs_time_and_no_result(impatient, case, warp, bar, parity):
    import ctypes

    from sbvr import _lib
    groups, per, shared, own, tps, nh, nkv, page = case
    c, q, pos, slots, starts = batch(*case, seed=31)
    sl, common, n = ints(slots), c.common(slots, starts), groups * per
    need = ctypes.c_size_t(0)
    cache = ctypes.cast(c._at, ctypes.POINTER(_lib.Pages))
    _lib.check(_lib.lib.sbvr_pages_attention_scratch_bytes(cache, n, tps, nh, groups, ctypes.byref(need)))
    scratch = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, float("nan"))
    assert impatient.pages_wait_that_runs_out(warp, bar, parity) == 0
    rc = impatient.sbvr_pages_attention_f16(cache, 0, q.data_ptr(), nh * D, sl.data_ptr(), pos.data_ptr(), starts.data_ptr(), common.data_ptr(), groups,
                                            out.data_ptr(), scratch.data_ptr(), need.value, n, tps, nh, D ** -0.5, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    close(out, attention(c, 0, q, pos, slots, nh), shared + own)


def test_refusals():
    from sbvr import _lib
    c, q, pos, slots, starts = batch(1, 4, 64, 20, 1, 8, 2, 16, seed=23)
    common = c.common(slots, starts)
    inv = torch.ones(64, device="cuda")
    qkv = torch.zeros((4, 12 * D), dtype=torch.float16, device="cuda")
    before = c.pool.clone()
    for call in (lambda: c.attention(1, q, pos, slots), lambda: c.attention(-1, q, pos, slots), lambda: c.attention(0, q[:, :-D], pos, slots),
                 lambda: c.attention(0, q, pos, slots, scale=0.0), lambda: c.attention(0, q, pos, slots, scale=float("nan")),
                 lambda: c.attention(0, q, pos, slots, scale=-0.1), lambda: c.rope_append(1, qkv, pos, inv, slots)):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: c.attention(0, q.float(), pos, slots), lambda: c.attention(0, q.cpu(), pos, slots), lambda: c.attention(0, q[:3], pos, slots),
                 lambda: c.attention(0, q, pos.long(), slots), lambda: c.attention(0, q, pos, slots, group_starts=starts),
                 lambda: c.attention(0, q, pos, slots, group_starts=starts[:1], shared=common), lambda: c.attention(0, q.t(), pos, slots),
                 lambda: c.attention(0, q, pos[:3], slots), lambda: c.attention(0, q, pos, slots, out=q[:2]), lambda: c.rope_append(0, qkv[:, :-8], pos, inv, slots),
                 lambda: c.rope_append(0, qkv, pos, inv[:-1], slots), lambda: c.reserve([0, 1], ints([1])), lambda: c.fork([0], [1, 2]),
                 lambda: c.common(slots, starts[:1]), lambda: c.free([9]), lambda: c.fork([0, 1], [2, 2]), lambda: c.reserve([0], -1), lambda: c.free([])):
        with pytest.raises((ValueError, TypeError)):
            call()
    lib, st = _lib.lib, torch.cuda.current_stream().cuda_stream
    out = torch.zeros_like(q)
    args = [c._at, 0, q.data_ptr(), 8 * D, None, pos.data_ptr(), None, None, 0, out.data_ptr(), None, 0, 4, 1, 8, 0.1, st]
    import ctypes

    def with_(i, v):
        a = list(args)
        a[i] = v
        return lib.sbvr_pages_attention_f16(ctypes.cast(a[0], ctypes.POINTER(_lib.Pages)), *a[1:])
    assert with_(12, 4) == 0 and with_(12, 0) == -1 and with_(14, 7) == -1 and with_(12, 6) == -1 and with_(3, 8 * D - 8) == -1
    assert with_(3, 8 * D + 1) == -3 and with_(2, q.data_ptr() + 2) == -3 and with_(5, None) == -1 and with_(8, 2) == -1
    torch.cuda.synchronize()
    assert torch.equal(c.pool.view(torch.int16), before.view(torch.int16))
    with pytest.raises(RuntimeError, match="no page"):           # (of the one call that was taken: it reads slot i for sequence i, and one of them is empty)
        c.check()


# ------------------------------------------------------------------ together
def tiny(seed=3, **kw):
    from models.sbvr_llama import LlamaConfig, SBVRLlamaForCausalLM
    return SBVRLlamaForCausalLM(LlamaConfig.preset("tiny"), device="cuda", max_batch=8, max_ctx=400, **kw).init_synthetic(seed)


@pytest.mark.parametrize("L,B,P,page", [(100, 5, 9, 16), (33, 1, 1, 32), (0, 3, 7, 16), (200, 8, 40, 64)])
def test_generate_shared(L, B, P, page):
    """A prefix once and prompts of uneven lengths: a captured step equals an eager one, and the logits are those of the dense cache (two fp16 layers,
    whose rotary embeddings round differently: 1e-2, the bound of this model's outputs)."""
    m = tiny()
    c = m.attach_pages(60, page, max_seqs=8)
    g = torch.Generator(device="cuda").manual_seed(L)
    prefix = torch.randint(0, 1024, (L,), device="cuda", generator=g)
    prompts = torch.randint(0, 1024, (B, P), device="cuda", generator=g)
    lens = [P] + [1 + (7 * i) % P for i in range(1, B)]
    got = m.generate_shared(prefix, prompts, 6, prompt_lengths=lens)
    assert got.shape == (B, 6)
    assert torch.equal(got, m.generate_shared(prefix, prompts, 6, prompt_lengths=lens, use_graph=False))
    assert torch.equal(got, m.generate_shared(prefix, prompts, 6, prompt_lengths=torch.tensor(lens)))
    assert not c.refs.any() and not c.lengths.any() and (c.table == -1).all()
    m.generate_shared(prefix, prompts, 1, prompt_lengths=lens)
    logits = m._bufs[("paged", B * P, B, B)].logits.double()
    for i in range(B):
        ids = torch.cat((prefix, prompts[i, :lens[i]]))[None]
        want = m.forward(ids)[0, -1].double()
        assert (logits[i] - want).norm() / want.norm() < 1e-2


def test_generate_shared_refuses_what_does_not_fit():
    m = tiny()
    ids = torch.zeros((2, 5), dtype=torch.long, device="cuda")
    with pytest.raises(RuntimeError, match="attach_pages"):
        m.generate_shared(ids[0], ids, 2)
    m.attach_pages(6, 16, max_seqs=2)
    for args in ((ids[0], ids[:, :0], 2), (ids[0], ids, 0), (ids[0], ids.repeat(2, 1), 2), (ids[0], ids, 92)):
        with pytest.raises(ValueError):
            m.generate_shared(*args)
    with pytest.raises(ValueError):
        m.generate_shared(ids[0], ids, 2, prompt_lengths=[5, 0])
    assert m.generate_shared(ids[0], ids, 2).shape == (2, 2)
    m.pages.reserve([1], 3)
    with pytest.raises(ValueError, match="already"):
        m.generate_shared(ids[0], ids, 2)
    m.pages.free([1])
    assert m.generate_shared(ids[0], ids, 2).shape == (2, 2)


def test_generate_shared_ignores_what_pads_a_prompt():
    """Rows padded with -1, -100, the largest id there is, and with ids of the vocabulary: the same tokens."""
    m = tiny()
    m.attach_pages(60, 16, max_seqs=8)
    g = torch.Generator(device="cuda").manual_seed(4)
    prefix = torch.randint(0, 1024, (37,), device="cuda", generator=g)
    prompts = torch.randint(0, 1024, (4, 9), device="cuda", generator=g)
    lens = [9, 1, 4, 8]
    want = m.generate_shared(prefix, prompts, 5, prompt_lengths=lens)
    for pad in (-1, -100, 2 ** 31 - 1):
        padded = prompts.clone()
        for i, n in enumerate(lens):
            padded[i, n:] = pad
        assert torch.equal(m.generate_shared(prefix, padded, 5, prompt_lengths=lens), want)
        with pytest.raises(ValueError, match="vocabulary"):
            m.generate_shared(prefix, padded, 5)


@pytest.mark.parametrize("case", [(1, 3, 0, 90, 1, 4, 2, 16), (1, 5, 0, 300, 6, 8, 2, 64), (1, 40, 700, 90, 1, 32, 8, 64), (1, 140, 640, 40, 1, 4, 4, 32),
                                  (1, 2, 200, 150, 100, 8, 2, 32)])
@pytest.mark.parametrize("exponent", [20, 23, 24, 25, 26, 27, 28, 29, 40, 60])
def test_scores_of_any_size(case, exponent):
    """Scores beyond what 24 bits hold to a whole number: the largest take all weight, evenly where several keys are the same.  Keys are multiples of one
    value, so scores are equal or apart by 2^-6 of the largest and more: every weight but theirs is zero, also in 64 bits."""
    groups, per, shared, own, tps, nh, nkv, page = case
    c, q, pos, slots, starts = batch(*case, seed=51)
    g = torch.Generator(device="cuda").manual_seed(exponent)
    q.zero_()
    q.view(-1, nh, D)[:, :, 5] = 16384.0
    keys = torch.randint(-64, 33, c.pool[0, 0, ..., 0].shape, device="cuda", generator=g)
    keys[torch.rand(keys.shape, device="cuda", generator=g) < 0.02] = 33
    c.pool[0, 0] = 0
    c.pool[0, 0, ..., 5] = keys.half()
    # scale: scores times log2(e) of up to 33 / 64 of 2^(exponent + 1)
    scale = 2.0 ** (exponent - 19) * 0.6931471805599453
    common = c.common(slots, starts)
    ref = attention(c, 0, q, pos, slots, nh, scale)
    for say in (dict(group_starts=starts, shared=common), {}):
        close(c.attention(0, q, pos, slots, scale=scale, **say), ref, shared + own)


@pytest.mark.parametrize("case", [(1, 3, 0, 90, 1, 4, 2, 16), (1, 5, 0, 300, 6, 8, 2, 64), (1, 40, 700, 90, 1, 32, 8, 64), (1, 140, 640, 40, 1, 4, 4, 32),
                                  (1, 2, 200, 150, 100, 8, 2, 32), (1, 60, 200, 150, 100, 8, 8, 32)])
def test_scores_of_minus_infinity(case):
    """Keys with infinities: no weight where other scores are finite, NaN where there is no other (zero over zero), zeros for a row without keys."""
    groups, per, shared, own, tps, nh, nkv, page = case
    c, q, pos, slots, starts = batch(*case, seed=61)
    q.view(-1, nh, D)[:, :, 5] = 1.0
    pos[tps if tps > 1 else 2] = -1                            # (a place without a token among others)
    some, none = slots[0], slots[1]
    for s, cut in ((some, 20), (none, None)):
        own_pages = [int(p) for p in c.table[s] if p >= 0 and c.refs[p] == 1]
        c.pool[0, 0, own_pages, ..., 5] = float("-inf")
        if cut and int(c.lengths[s]) > shared + 1:             # its last token's key is finite
            at = int(c.lengths[s]) - 1
            c.pool[0, 0, int(c.table[s, at // page]), :, at % page] = 0.25
    if shared:
        c.pool[0, 0, c.table[slots[0], :shared // page].long(), ..., 5] = float("-inf")
    ref = attention(c, 0, q, pos, slots, nh)
    common = c.common(slots, starts)
    for say in (dict(group_starts=starts, shared=common), {}):
        out = c.attention(0, q, pos, slots, **say)
        nan = torch.isnan(ref[0])
        assert nan.any() and torch.equal(torch.isnan(out), nan)
        close(out.masked_fill(nan, 0), tuple(x.masked_fill(nan, 0) for x in ref), shared + own)
        assert not out[pos < 0].any()


def test_a_token_for_each_of_65536_slots():
    """The largest cache's slots all at once, few and many positions each."""
    from models.pages import PagedCache
    n = 65536
    c = PagedCache(1, 1, n, page_size=16, max_seqs=n, max_pages=1)
    assert torch.equal(c.reserve(None, 1, tokens_per_seq=1), torch.zeros(n, dtype=torch.int32, device="cuda"))
    some = torch.arange(n, device="cuda", dtype=torch.int32) % 16
    got = c.reserve(None, some, tokens_per_seq=17).view(n, 17)
    want = 1 + torch.arange(17, device="cuda", dtype=torch.int32).expand(n, 17)
    assert torch.equal(got, torch.where(want <= some[:, None], want, torch.full_like(want, -1)))
    c.check()
    assert torch.equal(c.lengths, 1 + some) and (c.refs == 1).all()
    assert torch.equal(c.table.view(-1), torch.arange(n, device="cuda", dtype=torch.int32))
    c.reserve(None, 16)
    with pytest.raises(RuntimeError, match="beyond"):
        c.check()
    c.free(torch.arange(n, device="cuda", dtype=torch.int32))
    assert not c.refs.any() and not c.lengths.any() and (c.table == -1).all()
    c.check()


def test_generate_shared_beside_other_sequences():
    """Slots of others are left as they are; pages that they hold are not counted on."""
    m = tiny()
    c = m.attach_pages(20, 16, max_seqs=4)
    g = torch.Generator(device="cuda").manual_seed(8)
    prefix = torch.randint(0, 1024, (40,), device="cuda", generator=g)
    prompts = torch.randint(0, 1024, (2, 5), device="cuda", generator=g)
    want = m.generate_shared(prefix, prompts, 4)
    c.reserve([3], 16 * 16)
    book = c.book.clone()
    assert torch.equal(m.generate_shared(prefix, prompts, 4), want) and torch.equal(c.book, book)
    c.reserve([3], 1)
    with pytest.raises(ValueError, match="pages"):
        m.generate_shared(prefix, prompts, 4)
    c.free([3])
    assert torch.equal(m.generate_shared(prefix, prompts, 4, use_graph=False), want)


def test_generate_shared_for_more_prompts_than_a_fork_takes():
    """1030 prompts, ten different ones in turn: the same prompt, the same tokens and logits (every row of a batch goes through the same kernels)."""
    m = tiny()
    c = m.attach_pages(1200, 16, max_seqs=1030, max_pages=4)
    g = torch.Generator(device="cuda").manual_seed(8)
    prefix = torch.randint(0, 1024, (20,), device="cuda", generator=g)
    ten = torch.randint(0, 1024, (10, 3), device="cuda", generator=g)
    out = m.generate_shared(prefix, ten.repeat(103, 1), 3)
    logits = m._bufs["paged", 1030, 1030, 1030].logits.view(103, 10, -1).double()
    assert torch.equal(out, out[:10].repeat(103, 1))
    assert ((logits - logits[0]).norm(dim=-1) < 1e-2 * logits.norm(dim=-1)).all()
    assert (logits[0, 1:] - logits[0, :-1]).norm(dim=-1).min() > 1e-2 * logits[0].norm(dim=-1).max()
    assert not c.refs.any()


@pytest.mark.parametrize("L,B,P,page,new", [(100, 5, 9, 16, 22), (33, 1, 1, 32, 4), (0, 3, 7, 16, 12), (200, 8, 40, 64, 40), (64, 4, 1, 64, 3), (5, 2, 70, 16, 9)])
@pytest.mark.parametrize("use_graph", [True, False])
def test_steps_of_generate_shared_against_the_dense_cache(L, B, P, page, new, use_graph):
    """The logits of several steps, across pages' ends, are those of the dense model on the whole sequence: prefix, prompt and the tokens so far (1e-2, the bound
    of this model's outputs); the token is the dense one's where its lead is larger than two rows' worth of that."""
    m = tiny()
    m.attach_pages(100, page, max_seqs=8)
    g = torch.Generator(device="cuda").manual_seed(L + P)
    prefix = torch.randint(0, 1024, (L,), device="cuda", generator=g)
    prompts = torch.randint(0, 1024, (B, P), device="cuda", generator=g)
    lens = [P] + [1 + (5 * i) % P for i in range(1, B)]
    for k in sorted({2, 3, new // 2, new - 1, new} - {0, 1}):
        got = m.generate_shared(prefix, prompts, k, prompt_lengths=lens, use_graph=use_graph)
        logits = m._bufs["paged", B, B, B].logits.double()
        for i in range(B):
            ids = torch.cat((prefix, prompts[i, :lens[i]], got[i, :-1].long()))[None]
            want = m.forward(ids)[0, -1].double()
            assert (logits[i] - want).norm() < 1e-2 * want.norm(), (k, i)
            lead = want.topk(2).values
            if lead[0] - lead[1] > 2 * 1e-2 * want.norm():
                assert int(got[i, -1]) == int(want.argmax())
            assert int(got[i, -1]) == int(m._bufs["paged", B, B, B].logits[i].argmax())


def test_logits_of_padded_prompts():
    """The pad ids of test_generate_shared_ignores_what_pads_a_prompt, seen in the logits of the last step: the same bits."""
    m = tiny()
    m.attach_pages(60, 16, max_seqs=8)
    g = torch.Generator(device="cuda").manual_seed(4)
    prefix = torch.randint(0, 1024, (37,), device="cuda", generator=g)
    prompts = torch.randint(0, 1024, (4, 9), device="cuda", generator=g)
    lens, seen = [9, 1, 4, 8], []
    for pad in (None, -1, -100, 2 ** 31 - 1):
        padded = prompts.clone()
        for i, n in enumerate(lens):
            if pad is not None:
                padded[i, n:] = pad
        m.generate_shared(prefix, padded, 5, prompt_lengths=lens)
        seen.append(m._bufs["paged", 4, 4, 4].logits.clone())
    assert torch.isfinite(seen[0]).all() and all(torch.equal(s, seen[0]) for s in seen[1:])


def test_calls_that_wait_for_room_in_the_stream_let_other_threads_run():
    """A stream takes about a thousand launches ahead of the GPU; a call behind them waits in the driver, without the interpreter's lock."""
    import threading
    import time
    c, q, pos, slots, starts = batch(1, 3, 40, 9, 1, 4, 2, 16, seed=71)
    sl, common, nobody = ints(slots), c.common(slots, starts), ints([3])
    inv, qkv = torch.ones(64, device="cuda"), torch.zeros((3, 8 * D), dtype=torch.float16, device="cuda")
    calls = [lambda: c.free(nobody), lambda: c.reserve(nobody, 0), lambda: c.fork(nobody, nobody), lambda: c.compact(), lambda: c.common(sl, starts),
             lambda: c.rope_append(0, qkv, pos, inv, sl), lambda: c.attention(0, q, pos, sl)]
    for call in calls:
        call()
        torch.cuda.synchronize()
        done = threading.Event()

        def work():
            for _ in range(1500):
                call()
            done.set()
        torch.cuda._sleep(1_200_000_000)                       # 0.6 s
        t = threading.Thread(target=work)
        worst, last, begun = 0.0, time.perf_counter(), time.perf_counter()
        t.start()
        while not done.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            worst, last = max(worst, now - last), now
        t.join()
        assert last - begun > 0.3 and worst < 0.25, (calls.index(call), worst, last - begun)
        torch.cuda.synchronize()


# ------------------------------------------------------------------ when the shared pages are read in common
def wide_batch(*case, **kw):
    """The same batch in a cache whose table could hold far more than it does: what sharing can save is counted by what slots can hold."""
    from models.pages import PagedCache
    c, *rest = narrow_batch(*case, **kw)
    groups, per, _, _, _, _, nkv, page = case
    width = max(c.max_pages, (128 << 20) // (max(1, groups * (per - 1)) * page * nkv * 512) + 1)
    w = PagedCache(c.layers, c.n_kv, c.pages, page_size=page, max_seqs=c.max_seqs, max_pages=width)
    w.pool.copy_(c.pool), w.table[:, :c.max_pages].copy_(c.table), w.lengths.copy_(c.lengths), w.refs.copy_(c.refs)
    return (w, *rest)


narrow_batch = batch
FEW = [case for case in CASES if case[1] > 1 and case[4] * case[5] // case[6] < 64]


@pytest.mark.parametrize("again", [lambda case=case: test_attention(case) for case in FEW] +
                         [lambda a=a: test_growing_scores(tps=1, step=a) for a in (0.02, 0.7, 9.0)] +
                         [lambda a=a: test_what_lies_behind_a_sequence_does_not_matter(a) for a in ((1, 4, 200, 30, 6, 8, 2, 16), (2, 9, 640, 20, 1, 8, 2, 128))] +
                         [lambda a=a: test_values_that_are_not_finite_reach_the_tokens_that_see_them(tps=a, groups=True) for a in (1, 5, 6)] +
                         [lambda a=a: test_entries_that_name_no_page(entry=-1, case=a) for a in ((1, 5, 200, 20, 1, 8, 2, 16), (1, 4, 300, 40, 6, 8, 2, 16))] +
                         [lambda a=a: test_scores_of_any_size(exponent=a, case=(1, 5, 0, 300, 6, 8, 2, 64)) for a in (23, 27, 40)] +
                         [lambda a=a: test_scores_of_any_size(exponent=a, case=(1, 6, 200, 300, 6, 8, 2, 64)) for a in (23, 26, 27, 28, 40)] +
                         [lambda: test_scores_of_minus_infinity((1, 7, 300, 150, 3, 8, 2, 32)), lambda: test_rows_apart_and_scales(),
                          lambda: test_any_batch_order_and_groups(), lambda: test_many_groups(), lambda: test_a_far_layer()])
def test_small_batches_on_wide_tables(monkeypatch, again):
    """Shared pages of any size, read in common."""
    import sys
    monkeypatch.setattr(sys.modules[__name__], "batch", wide_batch)
    again()


@pytest.mark.parametrize("case,launches", [((1, 4, 256, 40, 1, 4, 2, 16), 1), ((1, 8, 1024, 40, 1, 32, 8, 64), 1), ((1, 16, 1024, 40, 1, 32, 8, 64), 1),
                                           ((1, 16, 2048, 40, 1, 32, 8, 64), 2), ((1, 64, 1024, 40, 1, 32, 8, 64), 2), ((16, 1, 2048, 40, 1, 32, 8, 64), 1),
                                           ((1, 16, 2048, 40, 15, 32, 8, 64), 2)])
def test_pages_are_read_in_common_where_that_pays(case, launches):
    from launched import kernels
    c, q, pos, slots, starts = batch(*case, seed=81)
    common, sl = c.common(slots, starts), ints(slots)
    names = kernels(lambda: c.attention(0, q, pos, sl, group_starts=starts, shared=common))
    assert len(names) == launches and "attention_own_kernel" in names[-1] and (launches == 1 or "attention_shared_kernel" in names[0])
    assert len(kernels(lambda: c.attention(0, q, pos, sl))) == 1


@pytest.mark.parametrize("kids", [1, 4, 6, 7, 15])
@pytest.mark.parametrize("share", [True, False])
def test_copies_by_heads_and_by_planes(kids, share):
    """64 to 2880 planes of pages to copy, three heads each: fewer than half the grid go head by head."""
    c, m = make(layers=32, n_kv=3, pages=2 + 3 * (kids + 1), max_seqs=kids + 1, seed=kids)
    c.reserve([0], 39), m.reserve([0], [39], 0)
    (c.fork if share else c.copy)([0] * kids, list(range(1, kids + 1)))
    m.fork([0] * kids, list(range(1, kids + 1)), share)
    same(c, m)
    gone = list(range(0, kids, 2))
    c.free(gone), m.free(gone)
    c.compact(), m.compact()
    same(c, m)


@pytest.mark.parametrize("exponent", [23, 27, 40])
def test_scores_of_any_size_in_whole_blocks(exponent):
    """Prompts of so many sequences that a CTA has all keys of its rows and writes the output itself."""
    test_scores_of_any_size((1, 60, 200, 150, 100, 8, 8, 32), exponent)
