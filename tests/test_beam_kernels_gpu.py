"""The kernels of a beam search alone, each against a plain implementation: the selection over beams and vocabulary (64 bits),
copies of state and of pages (bit for bit)."""
import math

import numpy as np
import pytest
import torch

from torchless_rs_b200.csrc import ops
from torchless_rs_b200.csrc.ops import KernelError

pytestmark = pytest.mark.gpu
PAGE = 64
F32_MAX = float(np.finfo(np.float32).max)


def _plain_select(logits: np.ndarray, scores: np.ndarray, n: int):
    """By sorting, in 64 bits: (values, beams, tokens)."""
    S, B = scores.shape
    V = logits.shape[1]
    values = np.full((S, n), -np.inf)
    beams, tokens = np.full((S, n), -1), np.full((S, n), -1)
    for s in range(S):
        found = []
        for b in range(B):
            if not scores[s, b] > -np.inf:
                continue
            x = np.nan_to_num(logits[s * B + b].astype(np.float64), nan=-np.inf, posinf=F32_MAX, neginf=-np.inf)
            if x.max() == -np.inf:
                continue
            with np.errstate(over="ignore"):
                lse = x.max() + np.log(np.exp(x - x.max()).sum())
            v = float(scores[s, b]) + (x - lse)
            for t in np.argsort(-v, kind="stable")[:n]:
                if v[t] > -np.inf:
                    found.append((-v[t], b, int(t)))
        for r, (v, b, t) in enumerate(sorted(found)[:n]):
            values[s, r], beams[s, r], tokens[s, r] = -v, b, t
    return values, beams, tokens


def _check_select(logits, scores, n):
    """Tolerance of the values: their rounding to 32 bits is at most 2^-24 of them; the logarithm of a row's sum is off by the relative
    error of the sum of those exps that run in 32 bits: an exponent to the base 2 of up to 2^5 (smaller results have no weight) is
    rounded by 2^-20 at most, which is ln 2 as much of the exp, and ex2 by 2^-22 of its result: together below 2^-20."""
    from torchless_rs_b200.sampling import BeamSelector
    dev = torch.device("cuda")
    lt = logits if torch.is_tensor(logits) else torch.from_numpy(logits).to(dev)
    v, b, t = BeamSelector(dev).select(lt, torch.from_numpy(scores).to(dev), n)
    pv, pb, pt = _plain_select(lt.cpu().numpy(), scores, n)
    v, b, t = v.cpu().numpy().astype(np.float64), b.cpu().numpy(), t.cpu().numpy()
    assert b.dtype == np.int32 and t.dtype == np.int32
    np.testing.assert_array_equal(b, pb)
    np.testing.assert_array_equal(t, pt)
    live = pb >= 0
    assert (v[~live] == -np.inf).all()
    assert (np.abs(v[live] - pv[live]) <= np.abs(pv[live]) * 2.0 ** -24 + 2.0 ** -20).all()


def _rand(rng, S, B, V, spread=2.0):
    return (rng.standard_normal((S * B, V)) * spread).astype(np.float32), \
        (-20.0 - 4.0 * rng.random((S, B))).astype(np.float32)


@pytest.mark.parametrize("S,B,V,n", [
    (1, 1, 1, 1), (1, 1, 2, 2), (1, 2, 3, 6), (2, 3, 5, 15), (1, 1, 129, 128), (3, 2, 255, 4), (1, 4, 256, 8), (2, 2, 257, 4),
    (1, 1, 1023, 1), (2, 5, 1024, 10), (1, 3, 1025, 17), (1, 16, 4099, 32), (2, 4, 8191, 33), (1, 2, 8193, 64), (1, 2, 32000, 65),
    (1, 1, 131072, 128), (4, 8, 32000, 16), (40, 8, 20001, 16), (2, 1, 262147, 5), (70, 16, 300, 16)])
@pytest.mark.parametrize("spread", [0.01, 3.0])
def test_select(S, B, V, n, spread):
    rng = np.random.default_rng(S * 1000 + B * 100 + V + n)
    _check_select(*_rand(rng, S, B, V, spread), n)


@pytest.mark.parametrize("S,B,V,n", [(1, 64, 2000, 128), (2, 32, 9000, 64), (1, 16, 40000, 32), (3, 40, 5000, 100), (1, 100, 300, 128),
                                     (1, 8, 140000, 128)])
@pytest.mark.parametrize("dead", [0, 1])
def test_select_of_more_candidates_than_threads_hold(S, B, V, n, dead):
    """Beams whose candidates are many, some beams without a score; all of one row above the others' too."""
    logits, scores = _rand(np.random.default_rng(S + B + V), S, B, V)
    if dead:
        scores[:, ::3] = -np.inf
        scores[:, 1] += 50.0
    _check_select(logits, scores, n)


@pytest.mark.parametrize("V", [7, 600, 9000, 40000])
def test_select_ties_go_to_the_lowest_beam_and_token(V):
    rng = np.random.default_rng(V)
    x = rng.integers(0, 3, (6, V)).astype(np.float32)       # rows of three values
    x[3] = x[0]                                             # beams that are alike, of equal scores
    scores = np.full((2, 3), -1.5, dtype=np.float32)
    _check_select(x, scores, min(24, 3 * V))
    _check_select(np.zeros((6, V), np.float32), scores, min(24, 3 * V))
    _check_select(np.full((6, V), -F32_MAX, np.float32), scores, min(24, 3 * V))


@pytest.mark.parametrize("V", [33, 700, 8192, 70000])
def test_select_entries_that_are_no_numbers_and_rows_without_any(V):
    rng = np.random.default_rng(V)
    x, scores = _rand(rng, 5, 3, V)
    x[rng.random(x.shape) < 0.3] = -np.inf
    x[rng.random(x.shape) < 0.2] = np.nan
    x[0] = -np.inf                     # a row that leaves nothing
    x[3:6] = np.nan                    # a sequence that leaves nothing
    x[6] = -np.inf                     # one entry alone
    x[6, V // 2] = 1.0
    x[9, 5], x[9, V - 1] = np.inf, np.inf
    scores[2, 0] = -np.inf
    scores[4, :] = -np.inf             # no beam at all
    scores[3, 1] = np.nan
    _check_select(x, scores, 12)


def test_select_beams_without_a_score_are_not_read():
    x, scores = _rand(np.random.default_rng(1), 2, 4, 5000)
    x[1] = np.inf
    scores[0, 1] = -np.inf
    _check_select(x, scores, 8)


@pytest.mark.parametrize("V,n", [(2000, 16), (2000, 30), (40000, 100), (140000, 16)])
def test_select_entries_that_bunch_in_few_groups(V, n):
    """More entries reach the bound than there is room for: candidates of neighbouring indices in all rows, the rest masked."""
    rng = np.random.default_rng(V + n)
    x = np.full((64, V), -np.inf, dtype=np.float32)
    for r in range(64):
        for first in range(0, V, 1024 * 32):
            at = first + 4 * np.arange(0, min(8192, V - first - 4) // 1024) * 256     # a thread's entries in every round of loads
            for e in range(4):
                x[r, at + e] = rng.standard_normal(len(at))
    _check_select(x, (-rng.random((16, 4))).astype(np.float32), n)
    y = np.full((64, V), -np.inf, dtype=np.float32)
    y[:, :min(V, 1500)] = rng.standard_normal((64, min(V, 1500)))
    _check_select(y, (-rng.random((16, 4))).astype(np.float32), n)


@pytest.mark.parametrize("V,n", [(5000, 16), (40000, 8), (140000, 16), (140000, 100)])
@pytest.mark.parametrize("order", ["rising", "falling", "the largest at the end", "the largest at the end, and NaN", "one value"])
def test_select_entries_in_an_order(V, n, order):
    rng = np.random.default_rng(V + n)
    logits, scores = _rand(rng, 2, 3, V)
    if order in ("rising", "falling"):
        logits.sort(axis=1)
        if order == "falling":
            logits = np.ascontiguousarray(logits[:, ::-1])
    elif order == "one value":
        logits[:] = 0.5
    else:
        logits[:, -3000:] += 30.0
        if "NaN" in order:
            logits[:, V // 2::97] = np.nan
    _check_select(logits, scores, n)


@pytest.mark.parametrize("V,n", [(40, 4), (5000, 2), (5001, 12), (40000, 16), (140001, 8), (9000, 100)])
@pytest.mark.parametrize("where", ["everywhere", "first tile", "later tile", "spread", "spread, and NaN", "rising, then infinite"])
def test_select_more_infinite_entries_than_are_asked_for(V, n, where):
    """Each counts as the largest finite number: the first `n` of a row come with the beam's own score, finite ones beside them do not;
    other beams of the sequence are as ever."""
    rng = np.random.default_rng(V + n)
    x, scores = _rand(rng, 3, 3, V)
    scores[0] = (-5.0, -30.0, -30.0)          # the infinite ones first
    scores[1] = (-5.0, -4.0, -6.0)            # and among the others' (these lie some nats below their beam's score)
    scores[2] = (-90.0, -5.0, -math.inf)      # and last
    for r in (0, 3, 4, 6):
        if where == "everywhere":
            x[r] = np.inf
        elif where == "first tile":
            x[r, 2:min(V, 2 + n + 1 + r)] = np.inf
        elif where == "later tile":
            x[r, -(n + 1 + r):] = np.inf
        elif where == "rising, then infinite":
            x[r].sort()
            x[r, V // 3::7] = np.inf
        else:
            x[r, rng.permutation(V)[:min(V, 3 * n + r)]] = np.inf
            if "NaN" in where:
                x[r, rng.permutation(V)[:V // 3]] = np.nan
    _check_select(x, scores, min(n, V))


@pytest.mark.parametrize("V,n", [(300, 8), (5000, 16), (20001, 24), (70000, 100)])
def test_select_zeros_of_either_sign_are_equal(V, n):
    rng = np.random.default_rng(V)
    x = np.where(rng.random((6, V)) < 0.5, np.float32(0.0), np.float32(-0.0))
    x[rng.random(x.shape) < 0.3] = -1.0
    x[0, :V // 2] = np.float32(-0.0)
    x[0, V // 2:] = np.float32(0.0)
    x[4] = np.float32(-0.0)
    _check_select(x, np.full((2, 3), -1.5, dtype=np.float32), n)


@pytest.mark.parametrize("V", [999, 4099, 9001, 9002, 9004, 50257, 70003])
@pytest.mark.parametrize("layout", ["contiguous", "a view of wider rows", "a view whose rows begin alike"])
def test_select_beams_that_are_alike(V, layout):
    """Beams of one sequence with the same logits and the same score: every token comes from the lower beam first, then from the other,
    wherever in memory their rows begin."""
    rng = np.random.default_rng(V)
    wide = {"contiguous": V, "a view of wider rows": V + 5, "a view whose rows begin alike": (V + 7) // 4 * 4}[layout]
    store = torch.from_numpy(rng.standard_normal((10, wide)).astype(np.float32) * np.float32(0.5)).cuda()
    x = store[:, wide - V:]
    x[1:4] = x[0].clone()                     # sequence 0: beams 0 to 3
    x[7], x[8] = x[5].clone(), x[5].clone()   # sequence 1: beams 0, 2 and 3
    scores = np.full((2, 5), -3.25, dtype=np.float32)
    for n in (8, 30, 100):
        _check_select(x, scores, n)


def test_select_peaked_rows_and_near_ties():
    """One entry holds nearly all weight, and candidates of other beams come within 1e-6 of each other."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((32, 3000)).astype(np.float32)
    x[np.arange(32), rng.integers(0, 3000, 32)] = 14.0
    scores = np.full((8, 4), -3.0, dtype=np.float32) - np.arange(4, dtype=np.float32) * np.float32(1e-6)
    _check_select(x, scores, 16)


@pytest.mark.parametrize("V", [4099, 131072, 262144])
@pytest.mark.parametrize("n", [1, 16])
@pytest.mark.parametrize("top", [0.0, 7.3, -250.7])
def test_select_rows_whose_weight_lies_below_the_bound(V, n, top):
    """`n` entries, and all others one height below them, so that nearly all exps run in 32 bits and are rounded alike: a row's logarithm is off
    by less than 2^-19 (beam_select.cu).  Scores near it, so that values are near zero and their own rounding hides nothing."""
    from torchless_rs_b200.sampling import BeamSelector
    dev = torch.device("cuda")
    for part in range(4):
        low = (np.float32(top) - np.linspace(0.02 + 3.4 * part, 3.4 * part + 3.4, 64)).astype(np.float32)
        high = np.float32(top)
        x = np.repeat(low[:, None], V, axis=1)
        x[:, 5:5 + 3 * n:3] = high
        lse = np.float64(high) + np.log(n + (V - n) * np.exp(low.astype(np.float64) - np.float64(high)))
        scores = (lse - np.float64(high)).astype(np.float32)[:, None]
        v, _, t = BeamSelector(dev).select(torch.from_numpy(x).to(dev), torch.from_numpy(scores).to(dev), n)
        want = scores[:, 0].astype(np.float64) + (np.float64(high) - lse)
        assert (t.cpu().numpy() == 5 + 3 * np.arange(n)).all()
        assert (np.abs(v.cpu().numpy().astype(np.float64) - want[:, None]) <= 2.0 ** -19 + np.abs(want[:, None]) * 2.0 ** -24).all()


@pytest.mark.parametrize("V,n", [(50, 12), (5000, 16), (20001, 33), (70000, 8), (70000, 100)])
@pytest.mark.parametrize("rows", [2, 600])
@pytest.mark.parametrize("case", ["scores", "infinite", "tiny"])
def test_select_sums_that_are_equal_though_logits_are_not(V, n, rows, case):
    """Sums so far from zero (or logits so near it) that different logits of a beam have the same sum in 64 bits: the larger logit comes
    first, of equal ones the lower token, whatever the number of rows (which says how a row is cut)."""
    from torchless_rs_b200.sampling import BeamSelector
    dev = torch.device("cuda")
    rng = np.random.default_rng(V + n)
    x = rng.standard_normal((2, V)).astype(np.float32)
    scores = np.array([[-30.0, -31.0]], dtype=np.float32)
    if case == "scores":
        x[:, ::3] = np.round(x[:, ::3])
        scores = np.array([[-1e30, -1e30]], dtype=np.float32)
    elif case == "infinite":
        x[0, rng.permutation(V)[:n // 2]] = np.inf
        x[1] = -np.inf
    else:
        x = (x * np.float32(1e-25)).astype(np.float32)
    order = np.argsort(-x, axis=1, kind="stable")[:, :n]
    top = [np.nan_to_num(x[b].astype(np.float64), posinf=F32_MAX, neginf=-np.inf) for b in range(2)]
    sums = [float(scores[0, b]) + (t - (t.max() + np.log(np.exp(t - t.max()).sum()) if t.max() > -np.inf else 0.0)) for b, t in enumerate(top)]
    found = sorted([(-sums[b][t], b, -top[b][t], int(t)) for b in range(2) for t in order[b] if sums[b][t] > -np.inf])[:n]
    S = rows // 2
    lt = torch.from_numpy(np.tile(x, (S, 1))).to(dev)
    _, b, t = BeamSelector(dev).select(lt, torch.from_numpy(np.tile(scores, (S, 1))).to(dev), n)
    want_b, want_t = torch.tensor([f[1] for f in found]), torch.tensor([f[3] for f in found])
    assert len(found) == n
    assert (b.cpu() == want_b).all() and (t.cpu() == want_t).all()


def test_select_strided_and_misaligned_rows():
    rng = np.random.default_rng(9)
    whole = torch.from_numpy(rng.standard_normal((12, 5003)).astype(np.float32)).cuda()
    scores = (-rng.random((3, 4))).astype(np.float32)
    for lo, hi in ((0, 5000), (1, 5001), (2, 4099), (3, 5003)):
        _check_select(whole[:, lo:hi], scores, 9)
    _check_select(whole[::2, 1:300], scores[:, :2].copy(), 5)


def test_select_same_result_again_on_another_stream_and_from_a_graph():
    from torchless_rs_b200.sampling import BeamSelector
    x, scores = _rand(np.random.default_rng(3), 4, 4, 30000)
    xt, st = torch.from_numpy(x).cuda(), torch.from_numpy(scores).cuda()
    sel = BeamSelector(torch.device("cuda"))
    want = [t.clone() for t in sel.select(xt, st, 8)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = sel.select(xt, st, 8)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = sel.select(xt, st, 8)
        graphs.append((g, got))
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for got in [other] + [got for _, got in graphs]:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("bad", ["cpu", "dtype", "shape", "n0", "n129", "n_all", "stride", "scores"])
def test_select_refusals(bad):
    from torchless_rs_b200.sampling import BeamSelector
    x, s, n = torch.zeros((4, 50), device="cuda"), torch.zeros((2, 2), device="cuda"), 4
    if bad == "cpu":
        x = x.cpu()
    elif bad == "dtype":
        x = x.bfloat16()
    elif bad == "shape":
        x = x[:3]
    elif bad == "n0":
        n = 0
    elif bad == "n129":
        n, x = 129, torch.zeros((4, 500), device="cuda")
    elif bad == "n_all":
        n = 101
    elif bad == "stride":
        x = torch.zeros((4, 100), device="cuda")[:, ::2]
    else:
        s = torch.zeros((2, 4), device="cuda")[:, ::2]
    with pytest.raises(KernelError):
        BeamSelector(torch.device("cuda")).select(x, s, n)


# ---- copies ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape,dtype", [((1, 2, 1), torch.int32), ((3, 5, 7), torch.bfloat16), ((2, 4, 16, 33), torch.float32),
                                         ((24, 9, 3, 1155), torch.bfloat16), ((2, 6, 16, 128, 128), torch.float32),
                                         ((4, 3, 5), torch.uint8), ((1, 300, 12), torch.float32), ((2, 3, 4100), torch.float32)])
def test_copy_slots(shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(shape[-1])
    st = torch.randint(0, 120, shape, generator=g, device="cuda").to(dtype)
    slots = shape[1]
    order = torch.randperm(slots, generator=g, device="cuda").tolist()
    k = slots // 2 if slots < 300 else 290
    dst, keep = order[:k], order[k:]
    src = [keep[i % max(1, len(keep) - 1)] for i in range(k)]       # the last of them is not read
    want = st.clone()
    want[:, dst] = want[:, src]
    ops.core_ops(torch.bfloat16).copy_slots(st, src, dst)
    assert torch.equal(st, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layers,heads,dim,vdim", [(1, 1, 16, 16), (3, 2, 64, 64), (2, 8, 128, 128), (2, 1, 576, 0), (2, 3, 48, 80),
                                                   (1, 2, 192, 128), (2, 1, 20, 0)])
def test_copy_pages(dtype, layers, heads, dim, vdim):
    g = torch.Generator(device="cuda").manual_seed(dim + vdim)
    pages, n = 2 * PAGE + 5, PAGE
    st = torch.randn((layers, pages * heads * PAGE * (dim + vdim)), generator=g, device="cuda").to(dtype)
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    dst, src, counts = order[:n], [order[n + i // 2] for i in range(n)], list(range(1, PAGE + 1))
    want = st.clone()
    keys = pages * heads * PAGE * dim
    k, v = want[:, :keys].view(layers, pages, heads, PAGE, dim), want[:, keys:].view(layers, pages, heads, vdim, PAGE)
    for s, d, c in zip(src, dst, counts):
        k[:, d, :, :c] = k[:, s, :, :c]
        if vdim:
            v[:, d, :, :, :c] = v[:, s, :, :, :c]
    ops.core_ops(dtype).copy_pages(st, pages, heads, dim, vdim, src, dst, counts)
    assert torch.equal(st, want)


def test_copies_of_many_pairs_take_several_launches():
    st = torch.arange(2 * 1000 * 3, dtype=torch.int32, device="cuda").view(2, 1000, 3)
    want = st.clone()
    src, dst = [7] * 600, list(range(300, 900))
    want[:, dst] = want[:, src]
    ops.core_ops(torch.float32).copy_slots(st, src, dst)
    assert torch.equal(st, want)
