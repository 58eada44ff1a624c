"""`SBVRLlamaForCausalLM.generate_shared` without a GPU: a cache in pages that keeps its books in plain Python (tests/pages_model.py) and a step that only
records what it is given."""
import pytest
import torch

from tests.pages_model import Model


class Cache:
    """What generate_shared uses of models.pages.PagedCache."""

    def __init__(self, pages=60, page_size=16, max_seqs=8, max_pages=40):
        self.m = Model(pages, page_size, max_seqs, max_pages, torch.zeros(1, 1, pages, 1, page_size, 1))
        self.pages, self.page_size, self.max_seqs, self.max_pages = pages, page_size, max_seqs, max_pages

    lengths = property(lambda self: torch.tensor(self.m.lengths, dtype=torch.int32))
    refs = property(lambda self: torch.tensor(self.m.refs, dtype=torch.int32))

    @staticmethod
    def _list(v, n=None):
        return v.tolist() if isinstance(v, torch.Tensor) else [v] * n if isinstance(v, int) else list(v)

    def reserve(self, slots, tokens, tokens_per_seq=0):
        slots = self._list(slots)
        return torch.tensor(self.m.reserve(slots, self._list(tokens, len(slots)), tokens_per_seq), dtype=torch.int32)

    def free(self, slots):
        self.m.free(self._list(slots))

    def fork(self, src, dst):
        assert 1 <= len(dst) <= 1024                           # (of one call of the library)
        self.m.fork(self._list(src), self._list(dst))

    def common(self, slots, starts):
        slots, starts = self._list(slots), self._list(starts)
        return torch.tensor([self.m.common(slots[a:b]) for a, b in zip(starts, starts[1:])], dtype=torch.int32)

    def check(self):
        bits, self.m.status = self.m.status, 0
        if bits:
            raise RuntimeError(f"status {bits}")


def model(monkeypatch, cache):
    """A tiny model whose steps note the ids and positions they are given and answer with the last ids, plus one."""
    from models.sbvr_llama import LlamaConfig, SBVRLlamaForCausalLM
    m = SBVRLlamaForCausalLM(LlamaConfig.preset("tiny"), device="cpu", max_batch=8, max_ctx=16)
    m.embed_tokens = torch.zeros((m.config.vocab_size, 1), dtype=torch.float16)
    m.pages, m.steps = cache, []

    def step(b, tokens_per_seq, last_only):
        m.steps.append((b.ids.clone(), b.positions.clone()))
        b.next_ids.fill_(len(m.steps))
    monkeypatch.setattr(m, "_forward_rows", step)
    monkeypatch.setattr(m, "_check", lambda: None)
    return m


@pytest.mark.parametrize("L,P", [(20, 5), (0, 4), (16, 1)])
def test_places_without_a_token_read_no_row_of_the_embedding(monkeypatch, L, P):
    """What stands behind a prompt's last token may be anything: -1, -100, an id behind the vocabulary."""
    m = model(monkeypatch, Cache())
    V = m.config.vocab_size
    lens = [P, max(1, P - 2), 1]
    prompts = torch.arange(3 * P).view(3, P) % V
    for i, n in enumerate(lens):
        prompts[i, n:] = torch.tensor([-1, -100, V, 2 ** 40])[:P - n]
    m.generate_shared(torch.arange(L), prompts, 3, prompt_lengths=lens, use_graph=False)
    assert len(m.steps) == (L > 0) + 3
    for ids, _ in m.steps:
        assert ((ids >= 0) & (ids < V)).all()
    ids, pos = m.steps[L > 0]
    for i, n in enumerate(lens):
        assert torch.equal(ids.view(3, P)[i, :n].long(), prompts[i, :n])
        assert pos.view(3, P)[i].tolist() == [L + j if j < n else -1 for j in range(P)]


@pytest.mark.parametrize("where", ["prefix", "prompt"])
@pytest.mark.parametrize("bad", [-1, 1024, 2 ** 32])
def test_ids_outside_the_vocabulary_are_refused(monkeypatch, where, bad):
    m = model(monkeypatch, Cache())
    assert m.config.vocab_size == 1024
    prefix, prompts = torch.arange(20), torch.arange(8).view(2, 4)
    (prefix if where == "prefix" else prompts.view(-1))[3] = bad
    with pytest.raises(ValueError, match="vocabulary"):
        m.generate_shared(prefix, prompts, 2, use_graph=False)
    assert not m.steps and not m.pages.refs.any()


def test_what_a_step_runs_on_changes_and_its_graphs_go(monkeypatch):
    """Graphs hold the addresses and the choice of kernels of the time they were captured at: none outlives a change of the all-reduces."""
    import models.comm
    m = model(monkeypatch, Cache())
    m._graph, m._shared_graph = "dense", (1, "in pages")
    m.set_pushed_allreduce(False)
    assert m._graph is None and m._shared_graph is None and m.pushed_allreduce is False
    for unavailable in (False, True):
        def comm(*a):
            if unavailable:
                raise RuntimeError("no peer mapping")
            return "block"
        monkeypatch.setattr(models.comm, "SymmetricAllReduce", comm)
        m.tp_group, m._graph, m._shared_graph = "group", "dense", (1, "in pages")
        assert m.enable_fused_allreduce() is not unavailable
        assert m._graph is None and m._shared_graph is None


def _bytes(m):
    held = [t for b in m._bufs.values() for t in list(vars(b).values()) + list(b.extra.get("paged", {}).values()) if isinstance(t, torch.Tensor)]
    return sum(t.untyped_storage().nbytes() for t in held)


def test_activations_of_earlier_calls_are_not_kept(monkeypatch):
    """A prefix's activations are 12 KB a token of this model: they live for the call, a batch of prompts' until the next call, a captured step's with it."""
    m = model(monkeypatch, Cache(pages=200, max_seqs=8, max_pages=100))
    most = 0
    for L, B, P in ((300, 3, 5), (301, 3, 6), (700, 2, 9), (16, 1, 16), (0, 8, 1), (1000, 3, 5)):
        m.generate_shared(torch.zeros(L, dtype=torch.long), torch.zeros((B, P), dtype=torch.long), 2, use_graph=False)
        assert set(m._bufs) == {("paged", B, B, B), ("paged", B * P, B, B)}
        most = max(most, _bytes(m))
    assert most < 60 * 20000
    m._shared_graph = (2, None)
    m._act_paged(2, 2, 2)
    step = m._bufs["paged", 2, 2, 2]
    for L, B, P in ((300, 3, 5), (2, 1, 2), (7, 2, 9), (9, 3, 1)):
        m.generate_shared(torch.zeros(L, dtype=torch.long), torch.zeros((B, P), dtype=torch.long), 1, use_graph=False)
        assert m._bufs["paged", 2, 2, 2] is step and len(m._bufs) <= 3
    m._drop_graphs()
    m.generate_shared(torch.zeros(9, dtype=torch.long), torch.zeros((3, 5), dtype=torch.long), 1, use_graph=False)
    assert set(m._bufs) == {("paged", 3, 3, 3), ("paged", 15, 3, 3)}


def test_activations_in_pages_have_no_scratch_of_the_dense_cache(monkeypatch):
    m = model(monkeypatch, Cache())
    dense = m._act(4, 4)
    assert dense.att_scratch is not None                       # (a step of four tokens splits the dense cache's keys)
    m.generate_shared(torch.zeros(9, dtype=torch.long), torch.zeros((4, 3), dtype=torch.long), 2, use_graph=False)
    assert m._act(4, 4) is dense
    assert all(b.att_scratch is None for key, b in m._bufs.items() if key[0] == "paged")


def test_pages_that_other_slots_hold_are_not_counted_on(monkeypatch):
    m = model(monkeypatch, Cache(pages=20, page_size=16, max_seqs=4, max_pages=20))
    prefix, prompts = torch.zeros(40, dtype=torch.long), torch.zeros((2, 5), dtype=torch.long)
    m.generate_shared(prefix, prompts, 4, use_graph=False)     # two pages in common, one more each
    m.steps.clear()
    m.pages.m.reserve([3], [16 * 17], 0)
    with pytest.raises(ValueError, match="pages"):
        m.generate_shared(prefix, prompts, 4, use_graph=False)
    assert not m.steps and sum(m.pages.m.refs) == 17 and not any(m.pages.m.lengths[:3]) and not m.pages.m.status
    m.pages.m.free([3]), m.pages.m.reserve([3], [16 * 16], 0)
    assert m.generate_shared(prefix, prompts, 4, use_graph=False).shape == (2, 4)


def test_what_earlier_calls_could_not_do_is_said_before_anything_is_run(monkeypatch):
    m = model(monkeypatch, Cache())
    prompts = torch.zeros((2, 5), dtype=torch.long)
    m.pages.reserve([0], 10 ** 6)
    with pytest.raises(RuntimeError, match="status 2"):
        m.generate_shared(prompts[0], prompts, 4, use_graph=False)
    assert not m.steps
    assert m.generate_shared(prompts[0], prompts, 4, use_graph=False).shape == (2, 4)


def test_more_prompts_than_a_fork_takes(monkeypatch):
    n = 1100
    m = model(monkeypatch, Cache(pages=n + 10, page_size=16, max_seqs=n, max_pages=3))
    out = m.generate_shared(torch.zeros(17, dtype=torch.long), torch.zeros((n, 2), dtype=torch.long), 2, use_graph=False)
    assert out.shape == (n, 2)
    assert m.steps[1][1].view(n, 2).tolist() == [[17, 18]] * n and m.steps[2][1].tolist() == [19] * n
    assert not m.pages.refs.any()


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_ids_of_any_whole_type(monkeypatch, dtype):
    m = model(monkeypatch, Cache())
    prompts = torch.arange(8, dtype=dtype).view(2, 4)
    m.generate_shared(torch.arange(20, dtype=dtype), prompts, 2, prompt_lengths=[4, 2], use_graph=False)
    assert m.steps[0][0].tolist() == list(range(20)) and m.steps[1][0].tolist() == [0, 1, 2, 3, 4, 5, 0, 0]
