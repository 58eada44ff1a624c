"""The paged cache's checks that need no GPU: descriptions that the library refuses before it launches anything."""
import ctypes

import pytest



def describe(**changes):
    from sbvr import _lib
    c = _lib.Pages(pool=1 << 20, table=1 << 21, lengths=1 << 22, refs=1 << 23, status=1 << 24, scratch=1 << 25, layers=2, pages=10, page=16, n_kv=2, head_dim=128,
                   max_seqs=4, max_pages=8)
    for k, v in changes.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("changes,rc", [
    (dict(pool=None), -1), (dict(table=None), -1), (dict(scratch=None), -1), (dict(layers=0), -1), (dict(pages=0), -1), (dict(n_kv=-1), -1),
    (dict(max_seqs=0), -1), (dict(max_pages=0), -1), (dict(page=48), -7), (dict(page=8), -7), (dict(page=512), -7), (dict(head_dim=64), -7),
    (dict(max_seqs=70000), -7), (dict(pages=1 << 27), -7), (dict(max_pages=1 << 27), -7), (dict(pool=(1 << 20) + 8), -3), (dict(refs=(1 << 23) + 4), -3),
    (dict(table=(1 << 21) + 2), -3)])
def test_descriptions_that_are_refused(changes, rc):
    from sbvr import _lib
    lib, c = _lib.lib, ctypes.byref(describe(**changes))
    n = ctypes.c_size_t(0)
    assert lib.sbvr_pages_free(c, 1 << 26, 1, None) == rc
    assert lib.sbvr_pages_reserve(c, 1 << 26, None, 1, 1, None, 0, None) == rc
    assert lib.sbvr_pages_fork(c, 1 << 26, 1 << 26, 1, 1, None) == rc
    assert lib.sbvr_pages_compact(c, None) == rc
    assert lib.sbvr_pages_common(c, None, 1, 1 << 26, 1, 1 << 26, None) == rc
    assert lib.sbvr_pages_rope_append_f16(c, 0, 1 << 26, 1 << 26, 1 << 26, 1.0, None, 1, 1, 4, 1 << 26, None) == rc
    assert lib.sbvr_pages_attention_f16(c, 0, 1 << 26, 512, None, 1 << 26, None, None, 0, 1 << 26, None, 0, 1, 1, 4, 1.0, None) == rc
    assert lib.sbvr_pages_attention_scratch_bytes(c, 1, 1, 4, 0, ctypes.byref(n)) == rc


def test_arguments_that_are_refused():
    from sbvr import _lib
    lib, c, x = _lib.lib, ctypes.byref(describe()), 1 << 26
    assert lib.sbvr_pages_free(c, x, 0, None) == -1 and lib.sbvr_pages_free(c, x, 5, None) == -1
    assert lib.sbvr_pages_reserve(c, x, None, -1, 1, None, 0, None) == -1 and lib.sbvr_pages_reserve(c, x, None, 1, 1, x, 0, None) == -1
    assert lib.sbvr_pages_fork(c, None, x, 1, 1, None) == -1 and lib.sbvr_pages_fork(c, x, x, 5, 1, None) == -1
    assert lib.sbvr_pages_fork(ctypes.byref(describe(max_seqs=2000)), x, x, 1025, 1, None) == -7
    assert lib.sbvr_pages_common(c, None, 1, None, 1, x, None) == -1 and lib.sbvr_pages_common(c, None, 0, x, 1, x, None) == -1
    rope = lambda **k: lib.sbvr_pages_rope_append_f16(c, *[k.get(n, d) for n, d in (       # noqa: E731
        ("layer", 0), ("qkv", x), ("pos", x), ("inv", x), ("s", 1.0), ("slots", None), ("seqs", 1), ("tps", 1), ("nh", 4), ("q", 2 * x))], None)
    assert rope(layer=2) == -1 and rope(layer=-1) == -1 and rope(seqs=0) == -1 and rope(seqs=5) == -1 and rope(qkv=x + 8) == -3 and rope(q=None) == -1
    assert rope(seqs=1 << 20, tps=1 << 12, slots=x) == -7
    assert rope(q=x) == -1 and rope(q=x + 2032) == -1 and rope(q=x - 1008) == -1      # rows in one another's place
    att = lambda **k: lib.sbvr_pages_attention_f16(c, *[k.get(n, d) for n, d in (          # noqa: E731
        ("layer", 0), ("q", x), ("pitch", 512), ("slots", None), ("pos", x), ("starts", None), ("shared", None), ("groups", 0), ("out", 2 * x), ("scratch", None),
        ("bytes", 0), ("seqs", 1), ("tps", 1), ("nh", 4), ("scale", 1.0))], None)
    for bad in (dict(layer=2), dict(q=None), dict(pos=None), dict(out=None), dict(seqs=0), dict(tps=0), dict(nh=3), dict(nh=0), dict(groups=-1), dict(groups=1),
                dict(groups=2, starts=x, shared=x), dict(pitch=504), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(seqs=5)):
        assert att(**bad) == -1, bad
    assert att(q=x + 8) == -3 and att(pitch=513) == -3 and att(out=x + 4) == -3 and att(scratch=x + 4) == -3
    assert att(seqs=1 << 20, tps=1 << 10, slots=x) == -7
    assert att(out=x) == -1 and att(out=x + 1008) == -1 and att(q=2 * x + 1008) == -1


@pytest.mark.parametrize("kw", [dict(head_dim=64), dict(page_size=48), dict(pages=0), dict(layers=0), dict(max_seqs=0), dict(max_seqs=70000), dict(pages=2 ** 26),
                                dict(max_pages=2 ** 25)])
def test_caches_that_cannot_be_made(kw):
    from models.pages import PagedCache
    with pytest.raises(ValueError):
        PagedCache(**{**dict(layers=1, n_kv=2, pages=4), **kw})


def test_no_cpu_path():
    from models.pages import PagedCache
    with pytest.raises(RuntimeError, match="no CPU path"):
        PagedCache(1, 2, 4, device="cpu")


def test_scratch_holds_what_the_calls_keep_there():
    from sbvr import _lib
    for pages, seqs in ((1, 1), (10, 4), (65536, 256), (33, 65536)):
        n = ctypes.c_size_t(0)
        assert _lib.lib.sbvr_pages_scratch_bytes(ctypes.byref(describe(pages=pages, max_seqs=seqs)), ctypes.byref(n)) == 0
        up = (pages + 3) // 4 * 4
        assert n.value >= 4 * max(4 + (seqs + 4) + pages, 4 + up + 3 * pages, 4 + 2 * up + 3 * pages)
