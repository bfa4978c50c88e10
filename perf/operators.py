"""What beam search asks of the device at every step, as plain data: the selection of the best continuations over
beams and vocabulary, the copies that let one sequence go on from another one's cache, and the attention of one new
token per beam over a paged cache whose leading pages the beams of a prompt share.

`run` computes a case in its plain form, elementary tensor operations in 32 bits or more, or, where `own` is true,
by the library's kernels."""
import math

import torch

own = False
DEVICE = "cuda:0"
PAGE = 64


# ---- the cases -------------------------------------------------------------------------------------------

def _select(seqs, beams, vocab, n, spread, dead=0, masked=0):
    """`dead`: of so many sequences' beams one has no score; `masked`: that share (in percent) of the entries is -inf."""
    return {"op": "select", "seqs": seqs, "beams": beams, "vocab": vocab, "n": n, "spread": spread, "dead": dead,
            "masked": masked}


def _slots(dtype, layers, slots, pairs, size):
    return {"op": "slots", "dtype": dtype, "layers": layers, "slots": slots, "pairs": pairs, "size": size}


def _pages(dtype, layers, pairs, kv_heads, dim, vdim):
    return {"op": "pages", "dtype": dtype, "layers": layers, "pairs": pairs, "kv_heads": kv_heads, "dim": dim,
            "vdim": vdim}


def _attend(dtype, seqs, beams, heads, kv_heads, dim, shortest, longest, new, window=0):
    """Prompts of `shortest` to `longest` tokens, up to `new` tokens generated since; `window` 0: all keys."""
    return {"op": "attend", "dtype": dtype, "seqs": seqs, "beams": beams, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "shortest": shortest, "longest": longest, "new": new, "window": window}


def listed():
    cases = {
        # the smallest call: two beams of one prompt, a test's vocabulary
        "select_1x2x256": _select(1, 2, 256, 4, 1.0),
        # a batch of prompts with four beams each at the 7B model's vocabulary
        "select_8x4x32000": _select(8, 4, 32000, 8, 2.5, dead=2),
        # the largest: many prompts, eight beams, the largest vocabulary
        "select_64x8x131072": _select(64, 8, 131072, 16, 2.0),
        # a recurrence's state in the layers of a model: half of the beams go on from another one
        "slots_f32_16x32": _slots("float32", 16, 32, 16, 16 * 128 * 128),
        # the last taps of short convolutions: rows of a few kilobytes, an odd number of them
        "slots_bf16_24x9": _slots("bfloat16", 24, 9, 3, 3 * 1155),
        # half filled last pages of a 7B model's layers, three of four beams of eight prompts
        "pages_bf16_32x24": _pages("bfloat16", 32, 24, 8, 128, 128),
        # the same in 32-bit, a small model
        "pages_f32_4x5": _pages("float32", 4, 5, 2, 64, 64),
        # interactive use: one prompt, four beams
        "attend_7b_1x4": _attend("bfloat16", 1, 4, 32, 8, 128, 2000, 2000, 20, window=4096),
        # a batch of unequal prompts
        "attend_7b_8x4": _attend("bfloat16", 8, 4, 32, 8, 128, 300, 4000, 120),
        # long prompts, eight beams, six query heads to a key's head (the 22B sizes)
        "attend_22b_4x8": _attend("bfloat16", 4, 8, 48, 8, 128, 6000, 16000, 250),
        # heads of 64, sixteen beams, a window that has left the prompts' first pages
        "attend_hd64_6x16": _attend("bfloat16", 6, 16, 16, 4, 64, 900, 3000, 130, window=1500),
        # the exact path: 32-bit keys and values
        "attend_f32_4x4": _attend("float32", 4, 4, 32, 8, 128, 500, 2000, 70),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "select", "slots", "pages", "attend", "attend", "attend"])
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        vocab = _log_int(rng, 200, 160000)
        seqs = _log_int(rng, 1, max(1, min(64, 60000000 // (beams * vocab))))
        return _select(seqs, beams, vocab, min(vocab, rng.choice([beams, 2 * beams, 3 * beams])), round(rng.uniform(0.7, 4.0), 3),
                       dead=rng.choice([0, 0, 1]) if beams > 1 else 0, masked=rng.choice([0, 0, 50]))
    if op == "slots":
        layers, slots, size = rng.randint(1, 24), rng.randint(2, 64), _log_int(rng, 1, 300000)
        slots = max(2, min(slots, 130000000 // (layers * size)))
        return _slots(rng.choice(["float32", "float32", "bfloat16"]), layers, slots, rng.randint(1, slots // 2), size)
    if op == "pages":
        dim = rng.choice([16, 32, 64, 128, 576])
        kv = 1 if dim == 576 else rng.choice([1, 2, 4, 8])       # 576: one latent vector per position
        return _pages(rng.choice(["float32", "bfloat16", "bfloat16"]), rng.randint(1, 32), rng.randint(1, 24), kv, dim,
                      0 if dim == 576 else rng.choice([dim, 64]))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    beams = rng.choice([2, 3, 4, 5, 8, 16])
    heads, kv, dim = rng.choice([(32, 8, 128), (32, 8, 128), (48, 8, 128), (16, 4, 128), (16, 4, 64), (8, 8, 64), (16, 1, 128)])
    most = 2000 if dtype == "float32" else 16000
    seqs = _log_int(rng, 1, 8)
    most = max(64, min(most, 300000000 // (seqs * beams * heads * dim)))
    a, b = sorted((_log_int(rng, 1, most), _log_int(rng, 1, most)))
    return _attend(dtype, seqs, beams, heads, kv, dim, a, b, _log_int(rng, 1, 300), window=rng.choice([0, 0, 4096, 777]))


# ---- inputs ----------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(1000003 * (seed % 1000003) + 17)


def _normal(g, shape, dtype):
    """N(0, 1), drawn in the type itself."""
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=g)


def _ints(g, lo, hi, n):
    return torch.randint(lo, hi, (n,), generator=g, device=DEVICE).tolist()


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "select":
        S, B, V = case["seqs"], case["beams"], case["vocab"]
        logits = _normal(g, (S * B, V), torch.float32).mul_(case["spread"])
        if case["masked"]:
            # tokens that may not come next
            gone = torch.randint(0, 100, (S * B, V), generator=g, device=DEVICE, dtype=torch.uint8) < case["masked"]
            logits.masked_fill_(gone, -math.inf)
        # what beams of a few dozen tokens have come to: some nats apart
        scores = -30.0 - 3.0 * torch.rand((S, B), generator=g, device=DEVICE)
        for s in range(min(case["dead"], S)):
            scores[s, B - 1] = -math.inf
        return dict(case, logits=logits, scores=scores)
    dtype = getattr(torch, case["dtype"])
    if op == "slots":
        storage = _normal(g, (case["layers"], case["slots"], case["size"]), dtype)
        order = torch.randperm(case["slots"], generator=g, device=DEVICE).tolist()
        dst = order[:case["pairs"]]
        keep = order[case["pairs"]:]
        src = [keep[i] for i in _ints(g, 0, len(keep), case["pairs"])]     # a beam may go on several times
        return dict(case, storage=storage, src=src, dst=dst)
    if op == "pages":
        n_pages = 2 * case["pairs"] + 3
        size = n_pages * case["kv_heads"] * PAGE * (case["dim"] + case["vdim"])
        storage = _normal(g, (case["layers"], size), dtype)
        order = torch.randperm(n_pages, generator=g, device=DEVICE).tolist()
        dst = order[:case["pairs"]]
        src = [order[case["pairs"] + i] for i in _ints(g, 0, n_pages - case["pairs"], case["pairs"])]
        return dict(case, storage=storage, n_pages=n_pages, src=src, dst=dst, counts=_ints(g, 1, PAGE, case["pairs"]))
    S, B, H, G, d = (case[k] for k in ("seqs", "beams", "heads", "kv_heads", "dim"))
    lo, hi = case["shortest"], case["longest"]
    prompts = _ints(g, lo, hi + 1, S)
    prompts[0] = hi
    if S > 1:
        prompts[1] = lo
    new = _ints(g, 1, case["new"] + 1, S)
    new[0] = case["new"]
    lens = [p + n for p, n in zip(prompts, new)]
    shared = [p // PAGE for p in prompts]                       # whole pages of the prompt
    width = max(-(-n // PAGE) for n in lens)
    total = sum(c + B * (-(-n // PAGE) - c) for c, n in zip(shared, lens))
    ids = torch.randperm(total, generator=g, device=DEVICE).tolist()
    table, at = [], 0
    window = case["window"]
    for c, n in zip(shared, lens):
        cols = -(-n // PAGE)
        first = max(0, n - window) // PAGE if window else 0     # pages before it have been given back
        common = ids[at:at + c]
        at += c
        for _ in range(B):
            row = common + ids[at:at + cols - c]
            at += cols - c
            table.append([-1] * first + row[first:] + [-1] * (width - cols))
    rows = S * B
    slot = torch.randperm(rows, generator=g, device=DEVICE)
    page_table = torch.empty((rows, width), dtype=torch.int32, device=DEVICE)
    page_table[slot] = torch.tensor(table, dtype=torch.int32, device=DEVICE)
    return dict(case, q=_normal(g, (rows, H * d), dtype).mul_(1.5), k_pages=_normal(g, (total, G, PAGE, d), dtype),
                v_pages=_normal(g, (total, G, d, PAGE), dtype), out=torch.zeros((rows, H * d), dtype=dtype, device=DEVICE),
                page_table=page_table, seq_slot=slot.to(torch.int32), scale=1.0 / math.sqrt(d), lens=lens, shared=shared,
                seq_len=torch.tensor([n for n in lens for _ in range(B)], dtype=torch.int32, device=DEVICE),
                group_start=torch.arange(0, rows + 1, B, dtype=torch.int32, device=DEVICE),
                group_pages=torch.tensor(shared, dtype=torch.int32, device=DEVICE))


# ---- the library's kernels -------------------------------------------------------------------------------

def _own(s):
    from torchless_rs_b200.csrc import ops
    op = s["op"]
    if op == "select":
        if "selector" not in s:
            from torchless_rs_b200.sampling import BeamSelector
            s["selector"] = BeamSelector(DEVICE)
        return s["selector"].select(s["logits"], s["scores"], s["n"])
    if op == "slots":
        ops.core_ops(s["storage"].dtype).copy_slots(s["storage"], s["src"], s["dst"])
        return s["storage"]
    if op == "pages":
        ops.core_ops(s["storage"].dtype).copy_pages(s["storage"], s["n_pages"], s["kv_heads"], s["dim"], s["vdim"], s["src"],
                                                    s["dst"], s["counts"])
        return s["storage"]
    if "attention" not in s:
        from torchless_rs_b200.csrc.attention_shared import SharedAttention
        from torchless_rs_b200.parts.runtime import Workspace
        s["attention"] = SharedAttention.get(s["q"].dtype, s["dim"])
        s["workspace"] = Workspace(torch.device(DEVICE))
    s["attention"].decode(s["q"], s["k_pages"], s["v_pages"], s["out"], s["seq_len"], s["seq_slot"], s["page_table"],
                          s["group_start"], s["group_pages"], s["heads"], s["kv_heads"], s["window"] or None, s["scale"],
                          s["workspace"], lens=s["lens"], shared=s["shared"], group_rows=s["beams"])
    return s["out"]


# ---- the plain forms -------------------------------------------------------------------------------------

def _plain_select(s):
    S, B, V, n = s["seqs"], s["beams"], s["vocab"], s["n"]
    # 64 bits: which candidate comes before which hangs on differences across rows
    x = torch.nan_to_num(s["logits"].double(), nan=-math.inf, posinf=torch.finfo(torch.float32).max, neginf=-math.inf)
    top = x.amax(1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    lse = top + (x - top).exp().sum(1, keepdim=True).log()
    v = torch.where(x == -math.inf, -math.inf, s["scores"].double().view(S * B, 1) + (x - lse)).view(S, B * V)
    border = v.topk(n, 1).values[:, -1:]
    above, equal = v > border, v == border
    kept = above | (equal & (equal.cumsum(1) <= n - above.sum(1, keepdim=True)))     # of equal ones the first
    at = kept.nonzero()[:, 1].view(S, n)
    value, order = v.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    none = value == -math.inf
    return value.float(), torch.where(none, -1, at // V).int(), torch.where(none, -1, at % V).int()


def _plain_pages(s):
    L, n, G, d, dv = s["layers"], s["n_pages"], s["kv_heads"], s["dim"], s["vdim"]
    keys = n * G * PAGE * d
    src, dst = (torch.tensor(s[k], device=DEVICE) for k in ("src", "dst"))
    seen = torch.arange(PAGE, device=DEVICE) < torch.tensor(s["counts"], device=DEVICE)[:, None]
    k = s["storage"][:, :keys].view(L, n, G, PAGE, d)
    k[:, dst] = torch.where(seen[None, :, None, :, None], k[:, src], k[:, dst])
    if dv:
        v = s["storage"][:, keys:].view(L, n, G, dv, PAGE)
        v[:, dst] = torch.where(seen[None, :, None, None, :], v[:, src], v[:, dst])
    return s["storage"]


def _plain_attend(s):
    rows, H, G, d = s["q"].shape[0], s["heads"], s["kv_heads"], s["dim"]
    table = s["page_table"][s["seq_slot"].long()].long().clamp_min(0)
    q = s["q"].float().view(rows, G, H // G, d)
    k = s["k_pages"][table].float().transpose(1, 2).reshape(rows, G, -1, d)
    v = s["v_pages"][table].float().permute(0, 2, 1, 4, 3).reshape(rows, G, -1, d)
    place = torch.arange(k.shape[2], device=DEVICE)
    length = s["seq_len"].long()[:, None]
    seen = place < length
    if s["window"]:
        seen &= place >= length - s["window"]
    scores = torch.where(seen[:, None, None, :], (q @ k.transpose(2, 3)) * s["scale"], -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True)).exp()
    out = (weights @ v) / weights.sum(-1, keepdim=True)
    s["out"].copy_(out.reshape(rows, H * d))
    return s["out"]


def run(state):
    if own:
        return _own(state)
    if state["op"] == "select":
        return _plain_select(state)
    if state["op"] == "slots":
        st = state["storage"]
        st[:, state["dst"]] = st[:, state["src"]]
        return st
    return _plain_pages(state) if state["op"] == "pages" else _plain_attend(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "select":
        entries = case["seqs"] * case["beams"] * case["vocab"]
        return {"bytes": 4 * entries + 12 * case["seqs"] * case["n"], "flops": 4 * entries}
    size = 2 if case["dtype"] == "bfloat16" else 4
    if op == "slots":
        return {"bytes": 2 * size * case["layers"] * case["pairs"] * case["size"], "flops": 0}
    if op == "pages":           # pages are half filled on average
        return {"bytes": size * case["layers"] * case["pairs"] * PAGE * case["kv_heads"] * (case["dim"] + case["vdim"]), "flops": 0}
    S, B = case["seqs"], case["beams"]
    # the prompts' and the new tokens' mean lengths as `prepare` draws them
    prompts = [case["longest"], case["shortest"]][:S] + [(case["longest"] + case["shortest"]) / 2] * max(0, S - 2)
    new = [case["new"]] + [(case["new"] + 1) / 2] * (S - 1)
    keys = pairs = 0
    for p, n in zip(prompts, new):
        seen = min(p + n, case["window"]) if case["window"] else p + n
        common = max(0, p // PAGE * PAGE - (p + n - seen))
        keys += common + B * (seen - common)
        pairs += B * seen
    return {"bytes": size * (keys * case["kv_heads"] * 2 * case["dim"] + 2 * S * B * case["heads"] * case["dim"]),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- the definitions in 64 bits --------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        values = []
        for i in range(case["seqs"]):
            of_beams = []
            for b in range(case["beams"]):
                row = s["logits"][i * case["beams"] + b].double()
                of_beams.append(float(s["scores"][i, b]) + torch.log_softmax(row, 0))
            values.append(torch.cat(of_beams).nan_to_num(nan=-math.inf, neginf=-math.inf).sort(descending=True).values[:case["n"]])
        return torch.stack(values), None, None
    if case["op"] != "attend":
        return None              # copies: nothing is computed
    B, H, G, d = (case[k] for k in ("beams", "heads", "kv_heads", "dim"))
    out = torch.empty((case["seqs"] * B, H, d), dtype=torch.float64, device=DEVICE)
    for r in range(out.shape[0]):
        n = s["lens"][r // B]
        first = max(0, n - case["window"]) if case["window"] else 0
        pages = s["page_table"][int(s["seq_slot"][r])].tolist()[first // PAGE:-(-n // PAGE)]
        k = torch.cat([s["k_pages"][p].double() for p in pages], 1)[:, first % PAGE:][:, :n - first]
        v = torch.cat([s["v_pages"][p].double() for p in pages], 2)[:, :, first % PAGE:][:, :, :n - first]
        for h in range(G):
            q = s["q"][r].double().view(G, H // G, d)[h]
            out[r, h * (H // G):(h + 1) * (H // G)] = torch.softmax(q @ k[h].T * s["scale"], 1) @ v[h].T
    return out.reshape(-1, H * d)
