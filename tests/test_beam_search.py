"""Beam search's decisions, followed with a scripted engine against a plain search over whole token lists, and the cache's side of
it: pages that several sequences hold, copies before a write, the order of slots (no device needed)."""
import math

import numpy as np
import pytest
import torch

from torchless_rs_b200 import cli
from torchless_rs_b200.cache import (PAGE, Cache, CacheCapacityError, CacheRollbackError, CacheStateError, PagedKVRequest,
                                     PagedLatentRequest, StateRequest)
from torchless_rs_b200.engine.beam import generate_beams, held_pages, plan_beam_batches
from torchless_rs_b200.engine.batch import RowGroups, layout_step


# ---- the search ------------------------------------------------------------------------------------------

def toy_logits(seq, vocab):
    """A language model: numbers that depend on the whole sequence."""
    h = 0
    for t in seq:
        h = (h * 1000003 + t + 1) % (1 << 61)
    return np.random.default_rng(h).standard_normal(vocab) * 1.5


class Logits:
    def __init__(self, rows, vocab):
        self.rows, self.shape = rows, (len(rows), vocab)


class ScriptedEngine:
    """Stands in for the engine: a slot holds its sequence's tokens."""

    def __init__(self, slots, vocab):
        self.vocab, self.seq, self.free = vocab, {}, list(range(slots))
        self.most, self.groups, self.forked = 0, [], 0

    def start_sequences(self, n):
        assert n <= len(self.free)
        got = [self.free.pop() for _ in range(n)]
        self.seq.update({s: [] for s in got})
        self.most = max(self.most, len(self.seq))
        return got

    def end_sequences(self, slots):
        for s in slots:
            del self.seq[s]
            self.free.append(s)

    def step(self, slots, tokens, want="last", groups=None):
        assert want == "last" and len(set(slots)) == len(slots) == len(tokens)
        if groups is not None:
            assert sum(groups) == len(slots) and all(len(t) == 1 for t in tokens)
            self.groups.append(list(groups))
        for s, t in zip(slots, tokens):
            self.seq[s] = self.seq[s] + list(t)
        return Logits([toy_logits(self.seq[s], self.vocab) for s in slots], self.vocab)

    def fork(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        self.forked += len(dst)
        for a, b in zip(src, dst):
            assert b in self.seq
            self.seq[b] = list(self.seq[a])

    def reorder(self, slots, parents):
        return Cache.reorder(self, slots, parents)      # the rule itself is the cache's


def log_softmax(x):
    return x - x.max() - math.log(np.exp(x - x.max()).sum())


def select(logits, scores, n):
    B = len(scores[0])
    out = ([], [], [])
    for s, of in enumerate(scores):
        found = []
        for b, c in enumerate(of):
            if c > -math.inf:
                lp = log_softmax(logits.rows[s * B + b])
                found += [(-(c + lp[t]), b, t) for t in range(logits.shape[1])]
        found = sorted(found)[:n]
        found += [(math.inf, -1, -1)] * (n - len(found))
        for k, sign in ((0, -1), (1, 1), (2, 1)):
            out[k].append([sign * f[k] for f in found])
    return out


def plain_search(prompt, vocab, max_tokens, beams, penalty, stop, early=False):
    """(score, tokens, stopped) of the hypotheses, best first: whole lists, one sequence at a time."""
    live, done = [(0.0, [])], []
    for step in range(max_tokens):
        found = []
        for rank, (lp, toks) in enumerate(live):
            x = log_softmax(toy_logits(prompt + toks, vocab))
            found += [(-(lp + x[t]), rank, t, toks) for t in range(vocab)]
        found.sort(key=lambda f: f[:3])
        nxt = []
        for neg, _, t, toks in found[:beams * (1 + len(stop))]:
            if t in stop:
                if len(nxt) < beams:
                    done.append((-neg / (len(toks) + 1) ** penalty, toks, True))
            elif len(nxt) < beams:
                nxt.append((-neg, toks + [t]))
        done = sorted(done, key=lambda d: -d[0])[:beams]
        live = nxt
        if not live:
            return done
        n = len(live[0][1])
        if n == max_tokens:
            done += [(lp / n ** penalty, toks, False) for lp, toks in live]
            return sorted(done, key=lambda d: -d[0])[:beams]
        if len(done) >= beams:
            best = live[0][0] / (max_tokens if penalty > 0 else n + 1) ** penalty
            if early or done[-1][0] >= best:
                return done
    return done


@pytest.mark.parametrize("beams", [1, 2, 3, 5])
@pytest.mark.parametrize("stop", [(), (3,), (0, 5)])
@pytest.mark.parametrize("penalty", [0.0, 1.0, 2.0, -0.5])
def test_search_equals_the_plain_one(beams, stop, penalty):
    vocab = 11
    prompts = [[1, 2, 3], [4], [9, 9, 9, 9, 9], [7, 1]]
    eng = ScriptedEngine(3 * beams, vocab)
    got = generate_beams(eng, select, prompts, 7, beams, penalty, stop, n_best=beams, cache_tokens=10 ** 6, max_batch=3 * beams)
    for p, r in zip(prompts, got):
        want = plain_search(p, vocab, 7, beams, penalty, set(stop))
        assert [h.tokens for h in r.hypotheses] == [t for _, t, _ in want]
        assert [h.stopped_at_eos for h in r.hypotheses] == [s for _, _, s in want]
        assert np.allclose([h.score for h in r.hypotheses], [s for s, _, _ in want])
        assert r.prompt_len == len(p) and r.tokens == want[0][1]
    assert not eng.seq and eng.most <= 3 * beams and all(set(g) == {beams} for g in eng.groups)


def test_early_stop_and_one_beam_is_greedy():
    vocab = 6
    for early in (False, True):
        eng = ScriptedEngine(8, vocab)
        (r,) = generate_beams(eng, select, [[2, 2]], 30, 4, 1.0, (1,), n_best=4, early_stop=early, cache_tokens=10 ** 6, max_batch=8)
        want = plain_search([2, 2], vocab, 30, 4, 1.0, {1}, early)
        assert [h.tokens for h in r.hypotheses] == [t for _, t, _ in want]
    eng = ScriptedEngine(1, vocab)
    (r,) = generate_beams(eng, select, [[5]], 9, 1, cache_tokens=10 ** 6, max_batch=1)
    seq = [5]
    for _ in range(9):
        seq.append(int(np.argmax(toy_logits(seq, vocab))))
    assert r.tokens == seq[1:] and r.steps == 8


def test_more_beams_than_first_tokens():
    """A vocabulary smaller than the beams: places without a beam run along and never win."""
    eng = ScriptedEngine(16, 3)
    (r,) = generate_beams(eng, select, [[1]], 4, 8, 1.0, (), n_best=8, cache_tokens=10 ** 6, max_batch=16)
    want = plain_search([1], 3, 4, 8, 1.0, set())
    assert [h.tokens for h in r.hypotheses] == [t for _, t, _ in want]


def test_arguments_that_are_refused():
    eng = ScriptedEngine(4, 5)
    for kw, why in ((dict(max_tokens=-1), "max_tokens"), (dict(beams=0), "beams"), (dict(beams=65, stop_ids=(1,)), "beams"),
                    (dict(n_best=5), "n_best"), (dict(n_best=0), "n_best"), (dict(length_penalty=math.nan), "penalty")):
        with pytest.raises(ValueError, match=why):
            generate_beams(eng, select, [[1]], **{**dict(max_tokens=2, beams=4, cache_tokens=999, max_batch=9), **kw})
    with pytest.raises(ValueError, match="empty"):
        generate_beams(eng, select, [[1], []], 2, 2, cache_tokens=999, max_batch=9)
    with pytest.raises(ValueError, match="slots"):
        generate_beams(eng, select, [[1]], 2, 5, cache_tokens=999, max_batch=4)
    with pytest.raises(ValueError, match="cache tokens"):
        generate_beams(eng, select, [[1] * 100], 2, 4, cache_tokens=200, max_batch=4)
    assert generate_beams(eng, select, [[1]], 0, 2)[0].hypotheses == [] and generate_beams(eng, select, [], 5, 2) == []
    assert len(eng.free) == 4


def test_slots_come_back_when_a_step_raises():
    eng = ScriptedEngine(4, 5)
    eng.step, step = None, eng.step

    def broken(slots, tokens, want="last", groups=None):
        if groups is not None:
            raise RuntimeError("no room")
        return step(slots, tokens, want)
    eng.step = broken
    with pytest.raises(RuntimeError, match="no room"):
        generate_beams(eng, select, [[1]], 5, 4, cache_tokens=999, max_batch=4)
    assert len(eng.free) == 4


def test_batches_fit_the_cache():
    assert held_pages(64, 1, 4) == 1 and held_pages(65, 1, 4) == 1 + 4 and held_pages(10, 1, 3) == 3
    assert held_pages(200, 100, 4) == 3 + 4 * 2
    assert plan_beam_batches([10, 10, 10], 5, 4, 100 * PAGE, 8) == [[0, 1], [2]]
    assert plan_beam_batches([10, 10, 10], 5, 4, 8 * PAGE, 100) == [[0, 1], [2]]


def test_command_line():
    o = cli.parse_args(["--beams", "4", "--length-penalty", "0.5", "dir", "1 2"])
    assert o["beams"] == 4 and o["length_penalty"] == 0.5
    assert cli.parse_args(["dir"])["beams"] is None
    for argv in (["--beams", "0", "d"], ["--beams", "2", "--temperature", "0.5", "d"], ["--beams", "2", "--top-k", "3", "d"],
                 ["--beams", "2", "--top-p", "0.3", "d"], ["--length-penalty", "1", "d"], ["--beams", "x", "d"]):
        with pytest.raises(cli.CliError):
            cli.parse_args(argv)


# ---- the cache -------------------------------------------------------------------------------------------

def _cache(requests=None, max_tokens=2048, slots=8):
    return Cache(requests or [PagedKVRequest(2, 16), PagedKVRequest(2, 16), StateRequest((3, 2))], max_tokens, slots, None,
                 torch.float32, "cpu")


def _write(c, slots, lens, tag):
    """Grows the sequences to `lens` and writes tag * 1000 + position at every new position (paged entries), tag (state)."""
    past = [c.length(s) for s in slots]
    c.prepare(slots, lens)
    for g in c.paged:
        for layer in g.layers:
            view = g.view(layer)
            for s, a, b, t in zip(slots, past, lens, tag):
                for j in range(a, b):
                    page = int(g.table_host[s, j // PAGE])
                    assert g.holders[page] == 1, "a page that others hold is written"
                    if hasattr(view, "pages"):
                        view.pages[page, j % PAGE] = t * 1000 + j
                    else:
                        view.k_pages[page, :, j % PAGE] = t * 1000 + j
                        view.v_pages[page, :, :, j % PAGE] = -(t * 1000 + j)
    for g in c.states:
        for s, t in zip(slots, tag):
            g.storage[:, s] = t
    c.commit(slots, lens)
    c.check()


def _read(c, slot, g, layer):
    view, n = g.view(layer), c.length(slot)
    first = g.first_live[slot] * PAGE
    out = []
    for j in range(first, n):
        page = int(g.table_host[slot, j // PAGE])
        assert int(g.table_dev[slot, j // PAGE]) == page
        if hasattr(view, "pages"):
            out.append(float(view.pages[page, j % PAGE].unique().item()))
        else:
            out.append(float(view.k_pages[page, :, j % PAGE].unique().item()))
            assert float(view.v_pages[page, :, :, j % PAGE].unique().item()) == -out[-1]
    return first, out


def _expect(c, slot, pieces):
    """pieces: (tag, from, to): who wrote which positions."""
    want = [t * 1000.0 + j for t, a, b in pieces for j in range(a, b)]
    for g in c.paged:
        for layer in g.layers:
            first, got = _read(c, slot, g, layer)
            assert got == want[first:]
    for g in c.states:
        assert (g.storage[:, slot] == pieces[-1][0]).all()


@pytest.mark.parametrize("requests", [None, [PagedLatentRequest(24), PagedKVRequest(1, 16, v_head_dim=8)],
                                      [PagedKVRequest(2, 16, window=100), PagedKVRequest(2, 16, window=100, keep_first=3)]])
@pytest.mark.parametrize("prompt", [1, 63, 64, 65, 200])
def test_forked_sequences_share_pages_and_write_their_own(requests, prompt):
    c = _cache(requests)
    a, b, d = c.acquire(3)
    _write(c, [a], [prompt], [1])
    held = [g.pool.held_count for g in c.paged]
    c.fork([a, a], [b, d])
    c.check()
    assert [g.pool.held_count for g in c.paged] == held and c.length(b) == c.length(d) == prompt
    assert c.common_columns([[a, b, d]]) == [-(-prompt // PAGE)]
    _write(c, [a, b, d], [prompt + 1] * 3, [1, 2, 3])
    # the begun page was copied for two of the three; a new page where the prompt had filled its last
    for g, h in zip(c.paged, held):
        assert g.pool.held_count == h + (3 if prompt % PAGE == 0 else 2)
    assert c.common_columns([[a, b, d]]) == [prompt // PAGE]
    for s, t in ((a, 1), (b, 2), (d, 3)):
        _expect(c, s, [(1, 0, prompt), (t, prompt, prompt + 1)])
    new = c.reorder([a, b, d], [1, 1, 0])
    assert new == [b, d, a]                  # b goes on in its slot and in that of the one nobody named
    _write(c, new, [prompt + 130] * 3, [5, 6, 7])
    for s, t, o in ((b, 5, 2), (d, 6, 2), (a, 7, 1)):
        _expect(c, s, [(1, 0, prompt), (o, prompt, prompt + 1), (t, prompt + 1, prompt + 130)])
    c.release([a, b])
    c.check()
    _expect(c, d, [(1, 0, prompt), (2, prompt, prompt + 1), (6, prompt + 1, prompt + 130)])
    c.release([d])
    assert all(g.pool.held_count == 0 and not g.holders.any() for g in c.paged)


def test_random_beams_against_plain_lists():
    rng = np.random.default_rng(0)
    for trial in range(6):
        c = _cache([PagedKVRequest(1, 16), PagedKVRequest(1, 16, window=90), StateRequest((2,))], 64 * 60, 10)
        slots = c.acquire(5)
        n = int(rng.integers(1, 130))
        _write(c, slots[:1], [n], [1])
        c.fork([slots[0]] * 4, slots[1:])
        pieces, tag = [[(1, 0, n)] for _ in slots], 1
        for step in range(40):
            parents = rng.integers(0, 5, 5).tolist()
            slots = c.reorder(slots, parents)
            pieces = [list(pieces[p]) for p in parents]
            more = int(rng.choice([1, 1, 1, 17, 64]))
            tags = list(range(tag + 1, tag + 6))
            tag += 5
            _write(c, slots, [n + more] * 5, tags)
            for q, t in zip(pieces, tags):
                q.append((t, n, n + more))
            n += more
            for s, q in zip(slots, pieces):
                _expect(c, s, q)
        c.release(slots)
        c.check()
        assert all(g.pool.held_count == 0 for g in c.paged)


def test_truncate_of_a_shared_sequence_leaves_the_other_alone():
    c = _cache([PagedKVRequest(2, 16)])
    a, b = c.acquire(2)
    _write(c, [a], [200], [1])
    c.fork([a], [b])
    c.truncate(b, 70)
    c.check()
    _write(c, [b], [75], [2])            # into a page that `a` holds too: a copy
    _expect(c, a, [(1, 0, 200)])
    _expect(c, b, [(1, 0, 70), (2, 70, 75)])
    c.reset(a)
    c.check()
    _expect(c, b, [(1, 0, 70), (2, 70, 75)])


def test_no_room_for_a_copy_changes_nothing():
    c = _cache([PagedKVRequest(1, 16)], max_tokens=3 * PAGE, slots=4)
    s = c.acquire(4)
    c.prepare(s[:1], [100])
    c.commit(s[:1], [100])
    c.fork([s[0]] * 3, s[1:])
    g = c.paged[0]
    before = (g.table_host.copy(), g.holders.copy(), g.pool.free_count)
    with pytest.raises(CacheCapacityError, match="needs 3 more"):
        c.prepare(s, [101] * 4)              # three copies, one page is free
    assert np.array_equal(before[0], g.table_host) and np.array_equal(before[1], g.holders) and before[2] == g.pool.free_count
    c.check()
    c.prepare(s[:1], [101])                  # one of them has room
    c.commit(s[:1], [101])
    c.check()


def test_forks_that_are_refused():
    c = _cache()
    a, b = c.acquire(2)
    for src, dst in (([a], [7]), ([7], [a]), ([a], [a]), ([a, a], [b, b]), ([a, b], [b, a]), ([a], [])):
        with pytest.raises(CacheStateError):
            c.fork(src, dst)
    for slots, parents in (([a, b], [0]), ([a, b], [0, 2]), ([a, b], [-1, 0]), ([a, a], [0, 1])):
        with pytest.raises(CacheStateError):
            c.reorder(slots, parents)
    c.fork([], [])
    assert c.reorder([a, b], [1, 0]) == [b, a] and c.reorder([], []) == []
    with pytest.raises(CacheRollbackError):
        c.prepare([a], [5])
        c.commit([a], [5])
        c.truncate(a, 3)


def test_step_arrays_are_laid_out_as_before_and_groups_behind_them():
    assert set(layout_step([3], [1], [0], [[5]], [[0]])) == {"tokens", "token_seq", "token_pos", "seq_slot", "seq_start", "seq_len",
                                                             "want_rows", "token_from"}
    g = RowGroups([4, 1], [200, 7], [3, 0])
    assert g.key() == ((4, 1), 256, 1) and g.key() == RowGroups([4, 1], [190, 7], [2, 0]).key()


@pytest.mark.parametrize("requests", [None, [PagedLatentRequest(24)], [PagedKVRequest(2, 16, window=100), PagedKVRequest(2, 16)]])
@pytest.mark.parametrize("have,wanted", [(0, 1), (64, 65), (64, 300), (70, 129), (70, 71), (128, 193)])
def test_a_fork_after_a_step_that_did_not_run_to_its_end(requests, have, wanted):
    """The table has grown and the length has not: the pages beyond the length stay the source's own."""
    c = _cache(requests)
    a, b, d = c.acquire(3)
    if have:
        _write(c, [a], [have], [1])
    c.prepare([a], [wanted])             # (and the step raises)
    c.check()
    c.fork([a, a], [b, d])
    c.check()
    assert all(g.n_cols[s] == -(-have // PAGE) for g in c.paged for s in (b, d))
    for s, t in ((a, 1), (b, 2), (d, 3)):
        _write(c, [s], [wanted], [t])
    for s, t in ((a, 1), (b, 2), (d, 3)):
        _expect(c, s, [(1, 0, have), (t, have, wanted)])
    c.prepare([a, b], [wanted + 100] * 2)
    new = c.reorder([a, b, d], [0, 0, 1])
    _write(c, new, [wanted + 70] * 3, [5, 6, 7])
    for s, t, o in zip(new, (5, 6, 7), (1, 1, 2)):
        _expect(c, s, [(1, 0, have), (o, have, wanted), (t, wanted, wanted + 70)])
    c.release([a, b, d])
    c.check()
    assert all(g.pool.held_count == 0 and not g.holders.any() for g in c.paged)


def test_the_check_refuses_a_shared_page_beyond_a_length():
    c = _cache([PagedKVRequest(2, 16)])
    a, b = c.acquire(2)
    _write(c, [a], [128], [1])
    c.fork([a], [b])
    c.check()
    c.lengths[b] = 64
    with pytest.raises(CacheStateError, match="beyond"):
        c.check()


def _state(c):
    return [(g.table_host.copy(), g.table_dev.clone(), g.holders.copy(), list(g.n_cols), list(g.first_live), g.pool.free_count) for g in c.paged], \
        [g.storage.clone() for g in c.states], list(c.lengths)


def _same(before, c):
    paged, states, lengths = _state(c)
    for x, y in zip(before[0], paged):
        assert all(np.array_equal(np.asarray(u), np.asarray(v)) for u, v in zip(x, y))
    return all(torch.equal(x, y) for x, y in zip(before[1], states)) and before[2] == lengths


@pytest.mark.parametrize("which", [0, 1])
def test_copies_that_are_refused_change_nothing(which, monkeypatch):
    """As where another device is the current one: the copies raise before anything is launched."""
    c = _cache([PagedKVRequest(2, 16), PagedKVRequest(2, 16, window=100), StateRequest((3, 2))])
    a, b, d = c.acquire(3)
    _write(c, [a], [90], [1])
    _write(c, [d], [40], [2])
    before = _state(c)

    def refuse(*args):
        raise RuntimeError("not on this device")
    monkeypatch.setattr(c.states[0], "fork", refuse)
    with pytest.raises(RuntimeError, match="not on this device"):
        c.fork([a, a], [b, d])
    c.check()
    assert _same(before, c)
    monkeypatch.undo()
    c.fork([a, a], [b, d])
    before = _state(c)
    monkeypatch.setattr(c.paged[which], "copy_pages", refuse)
    with pytest.raises(RuntimeError, match="not on this device"):
        c.prepare([a, b, d], [91, 150, 300])
    c.check()
    assert _same(before, c)
    monkeypatch.undo()
    _write(c, [a, b, d], [91, 150, 300], [1, 2, 3])
    for s, t, n in ((a, 1, 91), (b, 2, 150), (d, 3, 300)):
        _expect(c, s, [(1, 0, 90), (t, 90, n)])


def test_steps_of_sequences_that_were_never_forked_look_for_no_shared_pages(monkeypatch):
    """A step's host time for them is what it was: the pages' holders are looked at from a fork on, until the cache is empty."""
    c = _cache()
    looked = []
    for g in c.paged:
        monkeypatch.setattr(g, "writes_into_shared", lambda *a, of=type(g).writes_into_shared, g=g: looked.append(1) or of(g, *a))
    a, b = c.acquire(2)
    _write(c, [a, b], [70, 3], [1, 2])
    _write(c, [a, b], [71, 4], [1, 2])
    assert not looked
    c.fork([a], [b])
    _write(c, [a, b], [72, 72], [1, 2])
    assert looked
    c.release([a])
    _write(c, [b], [73], [2])
    assert len(looked) == 2 * len(c.paged)
    c.release([b])
    (a,) = c.acquire(1)
    _write(c, [a], [70], [1])
    _write(c, [a], [71], [1])
    assert len(looked) == 2 * len(c.paged)


@pytest.mark.parametrize("lens,max_tokens", [((64, 63), 1), ((128, 127, 126), 1), ((64, 63, 10), 3), ((200, 192, 190, 1), 40)])
def test_the_command_line_makes_room_for_every_prompt(lens, max_tokens, monkeypatch, tmp_path, capsys):
    """A prompt that ends inside a page may need more pages than a longer one: the cache holds all prompts' beams at once."""
    from types import SimpleNamespace
    from torchless_rs_b200 import api, config
    prompts, seen = [[7] * n for n in lens], {}

    class FakeModel:
        def generate_beams(self, prompts, max_tokens, beams, **kw):
            seen["batches"] = plan_beam_batches([len(p) for p in prompts], max_tokens, beams, seen["max_tokens"], seen["max_batch"])
            return [SimpleNamespace(tokens=[1]) for _ in prompts]

    def load(where, dtype, max_tokens, max_batch, max_seq_len):
        seen.update(max_tokens=max_tokens, max_batch=max_batch)
        return FakeModel()
    monkeypatch.setattr(config, "load_config", lambda where: SimpleNamespace(max_position_embeddings=4096, bos_token_id=1, eos_token_ids=()))
    monkeypatch.setattr(api, "load", load)
    text = " ; ".join(" ".join(str(t) for t in p) for p in prompts)
    assert cli.main(["--beams", "4", "--max-tokens", str(max_tokens), str(tmp_path), text]) == 0, capsys.readouterr().err
    assert seen["batches"] == [list(range(len(lens)))]


@pytest.mark.parametrize("penalty", [400.0, -400.0, 1e300])
def test_length_penalties_that_leave_the_range_of_numbers_are_refused(penalty):
    """16^400 is no number, 16^-400 is zero: refused before a sequence is started."""
    eng = ScriptedEngine(4, 5)
    with pytest.raises(ValueError, match="penalty"):
        generate_beams(eng, select, [[1]], 16, 4, penalty, cache_tokens=999, max_batch=4)
    assert len(eng.free) == 4
    for fine in (250.0, -250.0):
        assert generate_beams(eng, select, [[1]], 16, 4, fine, cache_tokens=999, max_batch=4)[0].hypotheses
    assert generate_beams(eng, select, [[1]], 1, 4, penalty, cache_tokens=999, max_batch=4)[0].hypotheses       # 1 to any power
