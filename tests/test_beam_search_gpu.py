"""Beam search through the public entry points, and the run of its operators together: sequences that go on from one another's
cache give what sequences fed alone give, in every design, and a search finds what a plain one finds."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import beralix_tiny
import dunesun_tiny
import fezolorn_tiny
import kikopel_tiny
import rupasun_tiny
import tovapel_tiny
from helpers_gpu import TinyModel, assert_close
from tiny import CONFIGS, make_model_dir, random_tokens, read_weights_numpy
from torchless_rs_b200.csrc import attention_shared, ops

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DESIGNS = {"kikopel": (kikopel_tiny.KModel, "P"), "dunesun": (dunesun_tiny.DModel, "A"), "tovapel": (tovapel_tiny.TModel, "P"),
           "rupasun": (rupasun_tiny.TModel, "P"), "fezolorn": (fezolorn_tiny.FModel, None), "beralix": (beralix_tiny.BModel, None)}


@pytest.fixture(autouse=True)
def shared_pages_are_read_together(monkeypatch):
    """These models are far too small for it to pay."""
    monkeypatch.setattr(attention_shared, "WORTH", {t: (0.0, 0.0) for t in attention_shared.WORTH})


def _design(name, dtype):
    make, cfg = DESIGNS[name]
    if cfg is None:
        cfg = sorted({"fezolorn": fezolorn_tiny, "beralix": beralix_tiny}[name].CONFIGS)[0]
    return make(cfg, dtype, seed=0, max_tokens=2048)


def _lineage(tm, vocab, prompt, parents_at, steps, rng, groups, forked):
    """Logits of every step of four sequences that begin with one prompt and take their own tokens; parents_at[i]: who goes on from whom
    before step i.  `forked`: by fork and reorder; else every sequence is fed alone what it has come to."""
    eng = tm.engine
    draws = rng.integers(0, vocab, (steps, 4))
    seqs = [list(prompt) for _ in range(4)]
    out = []
    if forked:
        slots = eng.start_sequences(4)
        eng.step(slots[:1], [prompt])
        eng.fork([slots[0]] * 3, slots[1:])
        for i in range(steps):
            if i in parents_at:
                slots = eng.reorder(slots, parents_at[i])
            out.append(eng.step(slots, [[int(t)] for t in draws[i]], groups=groups).float().cpu().numpy().copy())
            eng.cache.check()
        eng.end_sequences(slots)
        return np.stack(out)
    # alone: the same steps from the start for every stretch between two reorders
    start = 0
    stops = sorted(parents_at) + [steps]
    for stop in stops:
        if start in parents_at:
            seqs = [list(seqs[p]) for p in parents_at[start]]
        slots = eng.start_sequences(4)
        for s, q in zip(slots, seqs):
            eng.step([s], [q[:len(prompt)]])
        for k in range(len(prompt), len(seqs[0])):
            eng.step(slots, [[q[k]] for q in seqs])
        for i in range(start, stop):
            out.append(eng.step(slots, [[int(t)] for t in draws[i]]).float().cpu().numpy().copy())
            for q, t in zip(seqs, draws[i]):
                q.append(int(t))
        eng.end_sequences(slots)
        start = stop
    return np.stack(out)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["mistral A", "mistral C", "mistral D", "mistral F"] + list(DESIGNS))
def test_sequences_that_go_on_from_one_another_equal_sequences_fed_alone(name, dtype):
    """Without groups every kernel is the same and reads the same numbers: bit for bit."""
    tm = TinyModel(name[-1], dtype, seed=3, max_tokens=2048) if name.startswith("mistral") else _design(name, dtype)
    vocab = tm.engine.vocab_size
    rng = np.random.default_rng(5)
    prompt = random_tokens(rng, 61, vocab)
    parents_at = {2: [1, 1, 0, 1], 5: [3, 2, 1, 0], 7: [2, 2, 2, 2]}
    seed = int(rng.integers(1 << 30))
    want = _lineage(tm, vocab, prompt, parents_at, 10, np.random.default_rng(seed), None, False)
    got = _lineage(tm, vocab, prompt, parents_at, 10, np.random.default_rng(seed), None, True)
    assert np.array_equal(got, want)
    assert tm.engine.cache.slots.held_count == 0
    tm.engine.cache.check()
    tm.engine.check_kernels()


@pytest.mark.parametrize("name,dtype", [("D", "float32"), ("D", "bfloat16"), ("F", "float32"), ("F", "bfloat16")])
@pytest.mark.parametrize("length", [130, 63])
def test_rows_that_share_pages_equal_the_plain_implementation(name, dtype, length):
    """With groups: 70 steps (replayed from graphs, across a page's border), a reorder on the way, two prompts of unequal lengths; every
    row's logits against the plain implementation of its whole sequence."""
    cfg = dict(CONFIGS[name], sliding_window=None if length == 63 else CONFIGS[name]["sliding_window"])
    tm = TinyModel(name, dtype, seed=4, max_tokens=4096, cfg=cfg)
    eng, vocab = tm.engine, tm.engine.vocab_size
    rng = np.random.default_rng(length)
    prompts = [random_tokens(rng, length, vocab), random_tokens(rng, length + 70, vocab)]
    beams = [4, 3]
    slots = eng.start_sequences(7)
    heads = [slots[0], slots[4]]
    eng.prefill(heads, prompts)
    eng.fork([heads[0]] * 3 + [heads[1]] * 2, slots[1:4] + slots[5:])
    seqs = [list(prompts[0]) for _ in range(4)] + [list(prompts[1]) for _ in range(3)]
    before = ops.launch_counts().get("attn_shared", 0)
    checked = 0
    for i in range(70):
        if i in (3, 40):
            parents = [1, 1, 0, 3, 5, 5, 6]
            slots = eng.reorder(slots, parents)
            seqs = [list(seqs[p]) for p in parents]
        toks = random_tokens(rng, 7, vocab)
        logits = eng.step(slots, [[t] for t in toks], groups=beams)
        seqs = [q + [t] for q, t in zip(seqs, toks)]
        if i in (0, 1, 2, 3, 4, 39, 40, 41, 69):
            got = logits.float().cpu().numpy()
            ref = np.stack([tm.reference(q)[-1] for q in seqs])
            assert_close(got, ref, dtype, f"step {i}")
            checked += 1
    assert checked == 9 and ops.launch_counts()["attn_shared"] > before
    eng.end_sequences(slots)
    eng.cache.check()
    eng.check_kernels()


def test_the_grouped_mixers_of_other_designs_take_shared_pages():
    """Window attention over plain scores in another design (heads of 64 or 128 in bfloat16) takes the same kernel."""
    tm = rupasun_tiny.TModel("S", "bfloat16", seed=0, max_tokens=2048)
    eng, vocab = tm.engine, tm.engine.vocab_size
    rng = np.random.default_rng(1)
    prompt = random_tokens(rng, 140, vocab)
    outs = []
    before = ops.launch_counts().get("attn_shared", 0)
    for groups in (None, [4]):
        slots = eng.start_sequences(4)
        eng.step(slots[:1], [prompt])
        eng.fork([slots[0]] * 3, slots[1:])
        draw = np.random.default_rng(2)
        outs.append(np.stack([eng.step(slots, [[t] for t in random_tokens(draw, 4, vocab)], groups=groups).float().cpu().numpy()
                              for _ in range(6)]))
        eng.end_sequences(slots)
    assert ops.launch_counts().get("attn_shared", 0) > before
    rms = np.sqrt(((outs[0] - outs[1]) ** 2).mean()) / np.sqrt((outs[0] ** 2).mean())
    assert rms <= 2e-2           # the bound of that design's tests


def test_few_shared_keys_are_read_row_by_row(monkeypatch):
    monkeypatch.undo()
    tm = TinyModel("D", "bfloat16", seed=6, max_tokens=1024)
    eng = tm.engine
    slots = eng.start_sequences(2)
    eng.step(slots[:1], [random_tokens(np.random.default_rng(0), 130, eng.vocab_size)])
    eng.fork([slots[0]], [slots[1]])
    before = ops.launch_counts().get("attn_shared", 0)
    shared = eng.step(slots, [[1], [2]], groups=[2]).clone()
    assert ops.launch_counts().get("attn_shared", 0) == before
    eng.end_sequences(slots)
    slots = eng.start_sequences(2)
    eng.step(slots[:1], [random_tokens(np.random.default_rng(0), 130, eng.vocab_size)])
    eng.fork([slots[0]], [slots[1]])
    assert torch.equal(eng.step(slots, [[1], [2]]), shared)
    eng.end_sequences(slots)


def _plain_search(tm, prompt, max_tokens, beams, penalty, stop):
    """Whole sequences through the plain implementation; (score, log-probability, tokens) of the hypotheses, best first."""
    live, done = [(0.0, [])], []
    for _ in range(max_tokens):
        found = []
        for rank, (lp, toks) in enumerate(live):
            x = tm.reference(prompt + toks)[-1].astype(np.float64)
            x = x - x.max() - math.log(np.exp(x - x.max()).sum())
            found += [(-(lp + x[t]), rank, int(t), toks) for t in np.argsort(-x, kind="stable")[:2 * beams * (1 + len(stop))]]
        found.sort(key=lambda f: f[:3])
        nxt = []
        for neg, _, t, toks in found[:beams * (1 + len(stop))]:
            if t in stop:
                if len(nxt) < beams:
                    done.append((-neg / (len(toks) + 1) ** penalty, -neg, toks))
            elif len(nxt) < beams:
                nxt.append((-neg, toks + [t]))
        done = sorted(done, key=lambda d: -d[0])[:beams]
        live = nxt
        n = len(live[0][1])
        if n < max_tokens and len(done) >= beams and done[-1][0] >= live[0][0] / (max_tokens if penalty > 0 else n + 1) ** penalty:
            return done
    done += [(lp / max_tokens ** penalty, lp, toks) for lp, toks in live]
    return sorted(done, key=lambda d: -d[0])[:beams]


@pytest.mark.parametrize("name,beams,penalty", [("A", 3, 1.0), ("B", 4, 0.0), ("D", 4, 1.0), ("D", 2, 2.0)])
def test_search_in_32_bit_finds_what_a_plain_search_finds(name, beams, penalty):
    tm = TinyModel(name, "float32", seed=21, max_tokens=2048, max_batch=2 * beams)
    rng = np.random.default_rng(4)
    prompts = [random_tokens(rng, n, tm.cfg["vocab_size"]) for n in (5, 70, 23)]
    first = _plain_search(tm, prompts[1], 6, beams, penalty, set())
    stop = first[0][2][2]
    for stops in ((), (stop,)):
        got = tm.model.generate_beams(prompts, max_tokens=6, beams=beams, length_penalty=penalty, stop_ids=stops, n_best=beams)
        for p, r in zip(prompts, got):
            want = _plain_search(tm, p, 6, beams, penalty, set(stops))
            assert [h.tokens for h in r.hypotheses] == [t for _, _, t in want]
            # a logit is off by at most 5e-5 + 1e-4 |ref| (the package's bound) of logits below 1, its row's logarithm of the sum too
            assert np.allclose([h.logprob for h in r.hypotheses], [lp for _, lp, _ in want], atol=7 * 2 * 1.5e-4)
    assert tm.engine.cache.slots.held_count == 0
    tm.engine.cache.check()


@pytest.mark.parametrize("name", ["D", "F"])
def test_a_hypothesis_in_bfloat16_scores_what_its_tokens_score_alone(name):
    tm = TinyModel(name, "bfloat16", seed=2, max_tokens=4096)
    rng = np.random.default_rng(8)
    prompts = [random_tokens(rng, n, tm.cfg["vocab_size"]) for n in (200, 64, 131)]
    got = tm.model.generate_beams(prompts, max_tokens=40, beams=5, stop_ids=(), n_best=3)
    assert tm.engine.h2d_bytes() > 0
    for p, r in zip(prompts, got):
        assert len({tuple(h.tokens) for h in r.hypotheses}) == 3 and r.steps == 39
        assert [h.score for h in r.hypotheses] == sorted((h.score for h in r.hypotheses), reverse=True)
        for h in r.hypotheses:
            assert len(h.tokens) == 40 and abs(h.score - h.logprob / 40) < 1e-9
            x = tm.reference(p + h.tokens[:-1])[len(p) - 1:].astype(np.float64)
            x = x - x.max(1, keepdims=True)
            lp = (x - np.log(np.exp(x).sum(1, keepdims=True)))[np.arange(40), h.tokens].sum()
            # 2.5 % of the largest logit for any one, and as much for its row's logarithm of the sum
            assert abs(lp - h.logprob) <= 40 * 2 * 2.5e-2 * np.abs(tm.reference(p)).max()


def test_search_of_a_model_with_state_of_fixed_size():
    km = _design("kikopel", "float32")
    rng = np.random.default_rng(3)
    prompts = [random_tokens(rng, n, km.engine.vocab_size) for n in (9, 66)]
    got = km.model.generate_beams(prompts, max_tokens=5, beams=3, stop_ids=(), n_best=3)
    for p, r in zip(prompts, got):
        want = _plain_search(km, p, 5, 3, 1.0, set())
        assert [h.tokens for h in r.hypotheses] == [t for _, _, t in want]


def test_generation_after_a_search_is_what_it_was():
    tm = TinyModel("D", "bfloat16", seed=6, max_tokens=2048, max_batch=8)
    rng = np.random.default_rng(6)
    prompts = [random_tokens(rng, n, tm.cfg["vocab_size"]) for n in (70, 20)]
    want = [r.tokens for r in tm.model.generate(prompts, max_tokens=20, temperature=0.0, stop_ids=())]
    tm.model.generate_beams(prompts, max_tokens=20, beams=4, stop_ids=())
    assert [r.tokens for r in tm.model.generate(prompts, max_tokens=20, temperature=0.0, stop_ids=())] == want


@pytest.mark.parametrize("slots,beams", [(5, 5), (40, 8), (100, 33)])
def test_page_tables_reach_the_device_whichever_rows_change(slots, beams):
    from torchless_rs_b200.cache import Cache
    from torchless_rs_b200.cache.requests import PagedKVRequest, StateRequest
    c = Cache([PagedKVRequest(1, 16), PagedKVRequest(1, 16, window=90), StateRequest((3,))], 64 * 20 * slots, slots, None,
              dtype=torch.bfloat16, device=torch.device("cuda:0"))
    rng = np.random.default_rng(slots)
    held = np.asarray(c.acquire(slots))
    live = sorted(rng.permutation(held)[:beams].tolist())
    lens = [100] * beams
    c.prepare(live, lens)
    c.commit(live, lens)
    for _ in range(60):
        live = c.reorder(live, rng.integers(0, beams, beams).tolist())
        some = sorted(rng.permutation(beams)[:max(1, int(rng.integers(beams)))].tolist())
        lens = [c.length(s) for s in live]
        c.prepare([live[i] for i in some], [lens[i] + 1 for i in some])
        c.commit([live[i] for i in some], [lens[i] + 1 for i in some])
        c.check()
        for g in c.paged:
            assert np.array_equal(g.table_dev.cpu().numpy(), g.table_host)
    c.release(held.tolist())
    c.check()


def test_step_refuses_groups_that_do_not_fit():
    tm = TinyModel("D", "bfloat16", seed=6, max_tokens=1024)
    s = tm.engine.start_sequences(2)
    for groups in ([1], [3], [2, 0], [1, 1, 1]):
        with pytest.raises(ValueError, match="groups"):
            tm.engine.step(s, [[1], [2]], groups=groups)
    tm.engine.end_sequences(s)


def test_command_line_searches():
    d = make_model_dir(CONFIGS["D"], 11, torch.float32)
    run = lambda *a: subprocess.run([sys.executable, os.path.join(ROOT, "bin", "torchless"), *a], capture_output=True, text=True, timeout=600)
    r = run("--beams", "3", "--max-tokens", "5", "--dtype", "float32", d, "1 4 9 ; 7")
    assert r.returncode == 0, r.stderr
    import torchless_rs_b200 as tl
    m = tl.load(d, dtype="float32", max_tokens=1024)
    want = m.generate_beams([[1, 4, 9], [7]], max_tokens=5, beams=3, stop_ids=())
    assert [line.split() for line in r.stdout.strip().splitlines()] == [[str(t) for t in w.tokens] for w in want]
    r = run("--beams", "3", "--top-k", "2", d, "1")
    assert r.returncode == 1 and "--beams" in r.stderr
