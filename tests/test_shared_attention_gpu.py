"""Decode attention of rows that share leading pages, against a plain implementation in 64 bits."""
import math

import pytest
import torch

from torchless_rs_b200.csrc import ops
from torchless_rs_b200.csrc.attention_shared import SharedAttention
from torchless_rs_b200.csrc.ops import KernelError
from torchless_rs_b200.parts.runtime import Workspace

pytestmark = pytest.mark.gpu
PAGE = 64
DEV = "cuda"


class Setting:
    """Groups of `beams[g]` rows of length lens[g] whose tables agree in shared[g] columns; pages in random order, numbers that no row
    sees are `junk`."""

    def __init__(self, dtype, nh, nkv, hd, beams, lens, shared, window=None, seed=0, spread=1.5, junk=1e4, pages_more=3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.dtype, self.nh, self.nkv, self.hd, self.window = dtype, nh, nkv, hd, window
        self.beams, self.lens, self.shared = list(beams), list(lens), list(shared)
        rows = sum(beams)
        width = max(max(-(-n // PAGE) for n in lens), 1) + 1
        total = sum(min(c, -(-n // PAGE)) + b * max(0, -(-n // PAGE) - c) for b, n, c in zip(beams, lens, shared)) + pages_more
        ids = torch.randperm(total, generator=g, device=DEV).tolist()
        at, table = 0, []
        for b, n, c in zip(beams, lens, shared):
            cols = -(-n // PAGE)
            c = min(c, cols)
            first = max(0, n - window) // PAGE if window else 0
            common = ids[at:at + c]
            at += c
            for _ in range(b):
                row = common + ids[at:at + cols - c]
                at += cols - c
                table.append([-1] * first + row[first:] + [-1] * (width - cols))
        self.table = table
        slots = torch.randperm(rows + 2, generator=g, device=DEV)[:rows]
        self.page_table = torch.full((rows + 2, width), -1, dtype=torch.int32, device=DEV)
        self.page_table[slots] = torch.tensor(table, dtype=torch.int32, device=DEV)
        self.seq_slot = slots.to(torch.int32)
        self.row_len = [n for b, n in zip(beams, lens) for _ in range(b)]
        self.seq_len = torch.tensor(self.row_len, dtype=torch.int32, device=DEV)
        starts = [0]
        for b in beams:
            starts.append(starts[-1] + b)
        self.group_start = torch.tensor(starts, dtype=torch.int32, device=DEV)
        self.group_pages = torch.tensor(shared, dtype=torch.int32, device=DEV)
        self.q = (torch.randn((rows, nh * hd), generator=g, device=DEV) * spread).to(dtype)
        self.k = torch.randn((total, nkv, PAGE, hd), generator=g, device=DEV).to(dtype)
        self.v = torch.randn((total, nkv, hd, PAGE), generator=g, device=DEV).to(dtype)
        seen = torch.zeros((total, PAGE), dtype=torch.bool, device=DEV)
        for row, n in zip(table, self.row_len):
            for j in range(max(0, n - window) if window else 0, n):
                seen[row[j // PAGE], j % PAGE] = True
        self.k[~seen[:, None, :].expand(-1, nkv, -1)] = junk
        self.v.masked_fill_(~seen[:, None, None, :], junk)
        self.scale = 1.0 / math.sqrt(hd)
        self.ws = Workspace(torch.device(DEV))

    def run(self, **change):
        out = torch.full_like(self.q, 7.0)
        a = dict(q=self.q, k_pages=self.k, v_pages=self.v, out=out, seq_len=self.seq_len, seq_slot=self.seq_slot, page_table=self.page_table,
                 group_start=self.group_start, group_pages=self.group_pages, nh=self.nh, nkv=self.nkv, window=self.window, scale=self.scale,
                 workspace=self.ws, lens=self.lens, shared=self.shared, group_rows=max(self.beams))
        a.update(change)
        SharedAttention.get(self.dtype, self.hd).decode(**a)
        return a["out"]

    def plain(self):
        """(out, and the weighted sum of |v|), in 64 bits."""
        rows, G = len(self.table), self.nh // self.nkv
        out = torch.zeros((rows, self.nh, self.hd), dtype=torch.float64, device=DEV)
        mass = torch.zeros_like(out)
        self.largest = 0.0
        for r, (row, n) in enumerate(zip(self.table, self.row_len)):
            lo = max(0, n - self.window) if self.window else 0
            if n == 0:
                continue
            places = torch.arange(lo, n, device=DEV)
            page = torch.tensor(row, device=DEV)[places // PAGE]
            k, v = self.k[page, :, places % PAGE].double(), self.v[page, :, :, places % PAGE].double()     # [keys, nkv, hd]
            q = self.q[r].double().view(self.nkv, G, self.hd)
            score = torch.einsum("hgd,nhd->hgn", q, k) * self.scale
            self.largest = max(self.largest, score.abs().max().item())
            p = torch.softmax(score, -1)
            out[r] = torch.einsum("hgn,nhd->hgd", p, v).reshape(self.nh, self.hd)
            mass[r] = torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(self.nh, self.hd)
        return out.reshape(rows, -1), mass.reshape(rows, -1)

    def check(self, got=None):
        """bfloat16: a weight is rounded by at most 2^-8 of it, so the sum by 2^-8 of the weighted sum of |v|; the result by 2^-8 of
        it; 32-bit sums of at most 4096 terms and exponentials are off by less than 2^-12 of that sum together.  32 bits: a score is a
        sum of head size terms and one product more, each step rounded by at most 2^-24 of the largest |score| S there is, so off by
        e = (head size + 2) 2^-24 S; weights are then off by a factor of at most exp(e) either way, in the weighted sum and in the sum, 2 e
        together; sums of n <= 4096 weights add less than 2^-13 (2^-24 n^(1/2) and exp's own 2^-23)."""
        got = self.run() if got is None else got
        want, mass = self.plain()
        assert torch.isfinite(got).all()
        if self.dtype == torch.bfloat16:
            bound = mass * (2.0 ** -8 + 2.0 ** -12) + want.abs() * 2.0 ** -8 + 1e-30
        else:
            bound = mass * max(2.0 ** -13, 2 * (self.hd + 2) * 2.0 ** -24 * self.largest) + 1e-30
        over = ((got.double() - want).abs() / bound).max().item()
        assert over <= 1.0, over


HEADS = [(torch.bfloat16, 8, 2, 64), (torch.bfloat16, 8, 2, 128), (torch.float32, 8, 2, 64), (torch.float32, 8, 2, 128)]


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("lens,shared", [([1], [0]), ([64], [0]), ([65], [1]), ([64], [1]), ([129, 63], [1, 0]), ([200, 1000, 64, 7], [3, 15, 1, 0]),
                                         ([4000], [60]), ([300, 2500], [0, 30])])
@pytest.mark.parametrize("junk", [1e4, float("nan"), float("inf")])
def test_lengths_and_common_pages(dtype, nh, nkv, hd, lens, shared, junk):
    Setting(dtype, nh, nkv, hd, [4] * len(lens), lens, shared, seed=sum(lens), junk=junk).check()


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float32, 128)])
@pytest.mark.parametrize("nh,nkv", [(1, 1), (3, 1), (4, 2), (5, 5), (12, 2), (14, 2), (16, 1), (33, 3)])
@pytest.mark.parametrize("beams", [[1], [2, 3], [5, 1, 16]])
def test_heads_and_beams(dtype, hd, nh, nkv, beams):
    lens = [333, 130, 700][:len(beams)]
    Setting(dtype, nh, nkv, hd, beams, lens, [4, 1, 10][:len(beams)], seed=nh + len(beams)).check()


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("window", [1, 63, 64, 65, 200, 1000])
@pytest.mark.parametrize("junk", [1e4, float("nan")])
def test_windows(dtype, nh, nkv, hd, window, junk):
    Setting(dtype, nh, nkv, hd, [3, 4, 2], [500, 64, 1111], [6, 0, 16], window=window, seed=window, junk=junk).check()


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
def test_a_key_that_stands_out_on_either_side_of_every_border(dtype, nh, nkv, hd):
    """One key has a score far above the others: the last common one, the first of a row's own, the newest, the first in the window."""
    for j, window in ((0, None), (127, None), (128, None), (383, None), (399, None), (100, 300), (101, 300)):
        s = Setting(dtype, nh, nkv, hd, [4], [400], [6], window=window, seed=j)
        s.k[s.table[0][j // PAGE], :, j % PAGE] = (s.q[0, :hd] * 4).to(dtype) if j >= 400 - (window or 400) else float("nan")
        s.check()


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
def test_scores_that_grow_from_page_to_page(dtype, nh, nkv, hd):
    """Every page's scores lie far above the pages' before, by a few and by some hundred powers of two: references have to move."""
    for step in (3.0, 40.0, 150.0):
        s = Setting(dtype, nh, nkv, hd, [4, 2], [700, 200], [9, 1], seed=1)
        q = s.q.view(-1, nh, hd)
        q[:, :, 0] = 1.0
        q[1, :, 0] = -1.0                    # one row sees them fall
        s.k[:, :, :, 0] = 0.0
        for row in s.table:
            for c, page in enumerate(row):
                if page >= 0:
                    s.k[page, :, :, 0] = c * step / s.scale
        s.check()


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS + [(torch.bfloat16, 16, 1, 64), (torch.bfloat16, 16, 1, 128)])
@pytest.mark.parametrize("blocks", [1, 3])
@pytest.mark.parametrize("step", [3.0, 10.0, 20.0, 45.0, -10.0, -45.0])
def test_scores_that_grow_within_a_block(dtype, nh, nkv, hd, blocks, step, monkeypatch):
    """The same where one block sees many pages one after the other: references move, or weights leave their range."""
    from torchless_rs_b200.csrc import attention_shared
    monkeypatch.setattr(attention_shared, "_sm_count", lambda device: blocks)
    s = Setting(dtype, nh, nkv, hd, [4, 2], [1500, 200], [20, 1], seed=2)
    q = s.q.view(-1, nh, hd)
    q[:, :, 0] = 1.0
    q[1, :, 0] = -1.0
    q[2, 0, 0] = 0.0
    s.k[:, :, :, 0] = 0.0
    for row in s.table:
        for c, page in enumerate(row):
            if page >= 0:
                s.k[page, :, :, 0] = c * step / s.scale
    s.check()


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("blocks", [1, 148])
@pytest.mark.parametrize("far", [30.0, 70.0, 100.0, 300.0, -30.0, -100.0, float("nan"), float("inf"), float("-inf")])
def test_a_first_key_that_stands_out_in_pages_of_another_row(dtype, nh, nkv, hd, blocks, far, monkeypatch):
    """No common pages: the first key that a block sees is row 0's own, and lies far from what the other rows see."""
    from torchless_rs_b200.csrc import attention_shared
    monkeypatch.setattr(attention_shared, "_sm_count", lambda device: blocks)
    s = Setting(dtype, nh, nkv, hd, [4], [150], [0], seed=6)
    q = s.q.view(-1, nh, hd)
    q[:, :, 0] = 1.0
    s.k[:, :, :, 0] = 0.0
    s.k[s.table[0][0], :, 0, 0] = far / s.scale
    if math.isfinite(far):
        s.check()
        return
    got = s.run().view(4, nh, hd)
    want, mass = s.plain()
    assert torch.isfinite(got[1:]).all()
    bound = (mass * 2.0 ** -8 * 1.1 + want.abs() * 2.0 ** -8).view(4, nh, hd)[1:]
    assert ((got[1:].double() - want.view(4, nh, hd)[1:]).abs() <= bound).all()


def _check_far(s):
    """The bound of `Setting.check` for scores of some dozen: in bfloat16 too a score is a sum of head size products, each step
    rounded by at most 2^-24 of the largest |score| S, and scaled, so weights are off by a factor of at most exp((head size + 2) 2^-24 S) either
    way, in the weighted sum and in the sum."""
    got = s.run()
    want, mass = s.plain()
    scores = 2 * (s.hd + 2) * 2.0 ** -24 * s.largest
    if s.dtype == torch.bfloat16:
        bound = mass * (2.0 ** -8 + 2.0 ** -12 + scores) + want.abs() * 2.0 ** -8 + 1e-30
    else:
        bound = mass * max(2.0 ** -13, scores) + 1e-30
    assert torch.isfinite(got).all()
    over = ((got.double() - want).abs() / bound).max().item()
    assert over <= 1.0, over


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("blocks", [1, 148])
def test_weights_that_stay_in_range_while_their_sum_does_not(dtype, nh, nkv, hd, blocks, monkeypatch):
    """The first key that a block sees lies 78 to 90 below the others: from 2^127 / n on the sum of n weights overflows, a signed sum of
    weighted values need not."""
    from torchless_rs_b200.csrc import attention_shared
    monkeypatch.setattr(attention_shared, "_sm_count", lambda device: blocks)
    for seed, n, c in ((6, 150, 0), (7, 150, 2), (8, 260, 4)):
        s = Setting(dtype, nh, nkv, hd, [4], [n], [c], seed=seed)
        s.q.view(-1, nh, hd)[:, :, 0] = 1.0
        s.k[:, :, :, 0] = 0.0
        for half in range(156, 181):
            s.k[s.table[0][0], :, 0, 0] = -0.5 * half / s.scale
            _check_far(s)


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("blocks", [1, 2, 148])
@pytest.mark.parametrize("count", [64, 128, 256, 1000])
def test_many_keys_of_one_height_far_above_the_first(dtype, nh, nkv, hd, blocks, count, monkeypatch):
    """`count` keys 80 to 89 above those before them, with values of 0.1 and less: the sum of weights leaves its range before the weighted sum
    does, in one piece or where pieces are joined."""
    from torchless_rs_b200.csrc import attention_shared
    monkeypatch.setattr(attention_shared, "_sm_count", lambda device: blocks)
    for first in (1, 64, 200):
        n = first + count
        s = Setting(dtype, nh, nkv, hd, [3], [n], [(n - 1) // PAGE], seed=first, spread=0.3)
        s.v.mul_(0.05)
        s.q.view(-1, nh, hd)[:, :, 0] = 1.0
        s.k[:, :, :, 0] = 0.0
        place = torch.arange(first, n, device=DEV)
        page = torch.tensor(s.table, device=DEV)[:, place // PAGE]           # [rows, keys]
        for half in range(160, 179):
            s.k[page, :, place % PAGE, 0] = 0.5 * half / s.scale
            _check_far(s)


@pytest.mark.parametrize("dtype,nh,nkv,hd", [(torch.bfloat16, 1, 1, 64), (torch.bfloat16, 1, 1, 128), (torch.float32, 1, 1, 128)])
@pytest.mark.parametrize("high", [100.0, 111.0, 120.0])
def test_pieces_whose_references_say_little_of_their_weights(dtype, nh, nkv, hd, high, monkeypatch):
    """Two blocks.  The first has the common keys, 81 above the first of them; the second begins with a key of row 0's own, `high` above all
    that, and row 1's own keys lie 38 below that one: most of what row 1 sees is in the first block, whose reference is the lower by far."""
    from torchless_rs_b200.csrc import attention_shared
    monkeypatch.setattr(attention_shared, "_sm_count", lambda device: 2)
    monkeypatch.setattr(attention_shared, "PER_SM", {torch.bfloat16: 1, torch.float32: 1})
    s = Setting(dtype, nh, nkv, hd, [2], [8 * PAGE], [4], seed=12, spread=0.3)
    s.q.view(-1, nh, hd)[:, :, 0] = 1.0
    s.k[:, :, :, 0] = 0.0
    common, own0, own1 = s.table[0][:4], s.table[0][4:8], s.table[1][4:8]
    s.k[common, :, :, 0] = 81.0 / s.scale
    s.k[common[0], :, 0, 0] = 0.0
    s.k[own0, :, :, 0] = high / s.scale
    s.k[own1, :, :, 0] = (high - 38.0) / s.scale
    _check_far(s)


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
def test_scores_far_apart_and_scale(dtype, nh, nkv, hd):
    s = Setting(dtype, nh, nkv, hd, [4, 2], [700, 90], [9, 1], spread=0.2, seed=1)
    s.k.mul_(20.0)                           # scores of a few dozen: most weights are nothing
    s.check()
    s.scale = 0.0
    s.check()
    s.scale = -0.05
    s.check()


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
def test_values_of_a_rows_own_pages_that_are_no_numbers_stay_with_it(dtype, nh, nkv, hd):
    """One row's own keys and values are infinite or NaN: its result is no number, the others' are what they were."""
    for lens, shared, j in (([300], [2], 130), ([300], [2], 299), ([200], [3], 199), ([130], [0], 5)):
        s = Setting(dtype, nh, nkv, hd, [4] * len(lens), lens, shared, seed=j)
        clean = s.run()
        for bad in (float("nan"), float("inf")):
            t = Setting(dtype, nh, nkv, hd, [4] * len(lens), lens, shared, seed=j)
            t.v[t.table[1][j // PAGE], 0, 3, j % PAGE] = bad
            got = t.run().view(4, nh, hd)
            mine = got[1, :nh // nkv, 3]
            assert not torch.isfinite(mine).any() and (torch.isnan(mine).all() or bad == float("inf"))
            rest = got.clone()
            rest[1, :nh // nkv, 3] = clean.view(4, nh, hd)[1, :nh // nkv, 3]
            t.v.copy_(s.v)
            t.check(rest.view(4, -1))
            t.k[t.table[2][j // PAGE], 1, j % PAGE] = bad
            got = t.run().view(4, nh, hd)
            assert not torch.isfinite(got[2, nh // nkv:]).any()
            got[2, nh // nkv:] = clean.view(4, nh, hd)[2, nh // nkv:]
            t.k.copy_(s.k)
            t.check(got.view(4, -1))


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
def test_rows_of_length_zero_give_zero(dtype, nh, nkv, hd):
    s = Setting(dtype, nh, nkv, hd, [2, 3], [0, 77], [0, 1])
    got = s.run()
    assert (got[:2] == 0).all()
    s.check(got)


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
def test_rows_behind_the_last_group_and_groups_without_rows(dtype, nh, nkv, hd):
    s = Setting(dtype, nh, nkv, hd, [3, 2], [200, 330], [3, 4], seed=11)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    q = torch.cat([s.q, s.q[:2] * float("nan")])
    out = torch.full_like(q, 7.0)
    s.run(q=q, out=out, seq_len=i32(s.row_len + [10 ** 6, -1]), seq_slot=i32(s.seq_slot.tolist() + [10 ** 6, -5]),
          group_start=i32([0, 0, 3, 3, 5, 5]), group_pages=i32([0, 3, 100, 4, 0]), lens=[440, 200, 0, 330, 64], shared=[0, 3, 0, 4, 0])
    s.check(out[:5])
    assert (out[5:] == 7.0).all()


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
def test_every_way_of_cutting_gives_the_result(dtype, nh, nkv, hd, monkeypatch):
    from torchless_rs_b200.csrc import attention_shared
    s = Setting(dtype, nh, nkv, hd, [4, 3], [1000, 333], [12, 3], seed=8)
    for row_blocks, parts, blocks in ((1, 160, 148), (1, 2, 148), (2, 3, 148), (4, 20, 7), (1, 5, 1), (3, 160, 500), (1, 9, 33)):
        monkeypatch.setattr(attention_shared, "shared_plan", lambda *a, plan=(row_blocks, parts): plan)
        monkeypatch.setattr(attention_shared, "_sm_count", lambda device, blocks=blocks: blocks)
        s.check()


def test_a_call_that_does_not_say_that_pages_are_shared_gives_the_same():
    s = Setting(torch.bfloat16, 8, 2, 128, [4, 4], [700, 300], [10, 4], seed=2)
    s.check(s.run(group_pages=torch.zeros_like(s.group_pages), shared=[0, 0]))
    want = s.run()
    # fewer shared columns than the tables have in common
    s.check(s.run(group_pages=torch.tensor([3, 1], dtype=torch.int32, device=DEV), shared=[3, 1]))
    # and the same bits again, on another stream, and from two graphs that are replayed in turn
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = s.run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        out = torch.zeros_like(s.q)
        with torch.cuda.graph(graph):
            s.run(out=out)
        graphs.append((graph, out))
    for graph, _ in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in [other] + [out for _, out in graphs]:
        assert torch.equal(got, want)
    ops.check_kernel_errors()


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("window", [None, 200])
@pytest.mark.parametrize("begun", [([3, 130], [0, 2]), ([64, 1024], [1, 16]), ([1, 1], [0, 0])])
def test_a_recorded_call_is_right_for_lengths_that_came_later(dtype, nh, nkv, hd, window, begun):
    """Recorded at other lengths and common pages than it is replayed with; `bound` covers what the common pages come to."""
    s = Setting(dtype, nh, nkv, hd, [4, 3], [450, 1100], [6, 16], window=window, seed=3)
    lens, pages = s.seq_len.clone(), s.group_pages.clone()
    out = torch.full_like(s.q, 7.0)
    of = dict(out=out, lens=begun[0], shared=begun[1], bound=18)
    row_len = [min(n, m) for b, n, m in zip(s.beams, begun[0], s.lens) for _ in range(b)]
    s.seq_len.copy_(torch.tensor(row_len, dtype=torch.int32))
    s.group_pages.copy_(torch.tensor(begun[1], dtype=torch.int32))
    if window:                                        # (pages before the window are not in the tables)
        s.group_pages.copy_(pages)
        s.seq_len.copy_(lens)
    s.run(**of)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(**of)
    s.seq_len.copy_(lens)
    s.group_pages.copy_(pages)
    graph.replay()
    s.check(out)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_many_groups_and_the_same_result_as_row_by_row(dtype, hd):
    """Against the decode attention that reads every row's pages for itself."""
    s = Setting(dtype, 8, 4, hd, [4] * 9, [100 + 173 * i for i in range(9)], [1 + 2 * i for i in range(9)], seed=4, junk=0.0)
    got = s.run()
    out = torch.zeros_like(s.q)
    ops.core_ops(dtype).attn_generic(s.q, s.k, s.v, out, (s.seq_len - 1).contiguous(), torch.arange(36, dtype=torch.int32, device=DEV),
                                     s.seq_slot, s.page_table, 8, 4, hd, None, s.scale)
    s.check(got)
    s.check(out)


def test_offsets_beyond_32_bits():
    """A cache whose pages begin beyond 2^31 numbers."""
    hd, nkv, pages = 128, 8, 2 ** 31 // (8 * 64 * 128) + 40
    s = Setting(torch.bfloat16, 16, nkv, hd, [4], [300], [3], seed=5)
    k = torch.zeros((pages, nkv, PAGE, hd), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros((pages, nkv, hd, PAGE), dtype=torch.bfloat16, device=DEV)
    shift = pages - s.k.shape[0]
    k[shift:], v[shift:] = s.k, s.v
    far = torch.where(s.page_table >= 0, s.page_table + shift, s.page_table)
    s.check(s.run(k_pages=k, v_pages=v, page_table=far))


@pytest.mark.parametrize("bad", ["type", "cpu", "heads", "q shape", "pages", "lengths", "starts", "too long", "negative", "window", "groups", "table"])
def test_refusals(bad):
    s = Setting(torch.bfloat16, 8, 2, 64, [4, 4], [100, 300], [1, 4])
    change = {"type": dict(q=s.q.float()), "cpu": dict(q=s.q.cpu()), "heads": dict(nh=34), "q shape": dict(q=s.q[:, :256].contiguous()),
              "pages": dict(v_pages=s.v[1:]), "lengths": dict(seq_len=s.seq_len[:5]), "starts": dict(group_start=s.group_start[:2]),
              "too long": dict(lens=[100, 10000]), "negative": dict(shared=[-1, 0]), "window": dict(window=0), "groups": dict(group_rows=0),
              "table": dict(page_table=s.page_table.long())}[bad]
    with pytest.raises(KernelError):
        s.run(**change)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["q", "out"])
def test_tensors_that_begin_inside_16_bytes_are_refused(dtype, name):
    s = Setting(dtype, 8, 2, 64, [4, 4], [100, 300], [1, 4])
    inside = torch.zeros(s.q.numel() + 1, dtype=dtype, device=DEV)[1:].view(s.q.shape)
    with pytest.raises(KernelError):
        s.run(**{name: inside})


def test_sizes_without_a_kernel():
    assert SharedAttention.get(torch.bfloat16, 32) is None and SharedAttention.get(torch.float16, 64) is None
    assert not SharedAttention.get(torch.bfloat16, 64).takes(34, 2) and SharedAttention.get(torch.float32, 64).takes(64, 2)
