"""Serving operators over a paged key-value cache: the append with the position rotation, the attention
of the newest rows of each sequence over the pages, and the attention over packed whole prompts.

Together they are the attention half of a layer when several sequences are served at once: a prompt
step rotates and appends its keys and values and attends over the packed prompts; a decode or a
speculative verify step appends one or a few rows a sequence and attends over the pages.  Activations
are float32 where they come from the quantised matmuls, or 16 bits; the cache holds float32, float16
or bfloat16.  Head layouts are those of the package's own configurations (1B: 32/8 heads of 64; 3B:
24/8 of 128; 8B: 32/8 of 128; 70B: 64/8 of 128) or generic.

The definition, for a sequence whose cache holds ``len`` positions after its n new rows: row i stands
at position p = len - n + i, is rotated by the angles of p in pairs (2j, 2j + 1), and attends over the
positions 0..p: out = sum_j softmax_j(scale * q.k_j) v_j.  A row that sees nothing answers zeros.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BASE = 500000.0


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one decode row of an 8B model into a float32 cache: pure latency, once a layer and token
        {"name": "append_1", "op": "append", "heads": 32, "kv": 8, "hd": 128, "type": "f32", "cache": "f32", "page": 16, "seqs": 1, "len": 700, "rows": 1},
        # a verify step of 48 sequences, up to five rows each, of a 70B model into a 16-bit cache
        {"name": "append_48x5", "op": "append", "heads": 64, "kv": 8, "hd": 128, "type": "f32", "cache": "bf16", "page": 64, "seqs": 48, "len": 900, "rows": 5},
        # four packed prompts of an 8B model, their rotated keys kept for the prompt attention
        {"name": "append_prompts", "op": "append", "heads": 32, "kv": 8, "hd": 128, "type": "f32", "cache": "f16", "page": 32, "seqs": 4, "len": 2711, "rows": 2711},
        # one chat of a 1B model, a few hundred positions: the smallest attention call
        {"name": "decode_1x300", "op": "paged", "heads": 32, "kv": 8, "hd": 64, "type": "f32", "cache": "f32", "page": 16, "seqs": 1, "len": 300, "rows": 1},
        # one very long document of an 8B model: few rows, so the positions are what is split
        {"name": "decode_1x15000", "op": "paged", "heads": 32, "kv": 8, "hd": 128, "type": "f32", "cache": "f16", "page": 16, "seqs": 1, "len": 15000, "rows": 1},
        # a speculative verify step of 16 sequences of an 8B model, up to five rows each, ragged lengths
        {"name": "verify_16x5", "op": "paged", "heads": 32, "kv": 8, "hd": 128, "type": "f32", "cache": "f32", "page": 24, "seqs": 16, "len": 3000, "rows": 5},
        # a full decode batch of a 70B model in 16 bits throughout: the cache's bytes are all that counts
        {"name": "decode_48x8000", "op": "paged", "heads": 64, "kv": 8, "hd": 128, "type": "bf16", "cache": "bf16", "page": 64, "seqs": 48, "len": 8000, "rows": 1},
        # a short question to a 1B model
        {"name": "prompt_1x37", "op": "packed", "heads": 32, "kv": 8, "hd": 64, "type": "f32", "seqs": 1, "len": 37},
        # several ragged prompts of a 3B model, float32 as the quantised matmuls leave them
        {"name": "prompt_6x1200", "op": "packed", "heads": 24, "kv": 8, "hd": 128, "type": "f32", "seqs": 6, "len": 1200},
        # many short ragged prompts of a 1B model in 16 bits
        {"name": "prompt_24x700", "op": "packed", "heads": 32, "kv": 8, "hd": 64, "type": "f16", "seqs": 24, "len": 700},
        # one long prompt of an 8B model, float32
        {"name": "prompt_1x4096", "op": "packed", "heads": 32, "kv": 8, "hd": 128, "type": "f32", "seqs": 1, "len": 4096},
        # one very long prompt of an 8B model in 16 bits: matrix products all the way
        {"name": "prompt_1x8192", "op": "packed", "heads": 32, "kv": 8, "hd": 128, "type": "bf16", "seqs": 1, "len": 8192},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "paged", "paged", "packed", "packed"])
    heads, kv, hd = rng.choice([(32, 8, 64), (24, 8, 128), (32, 8, 128), (64, 8, 128), (16, 16, 64), (12, 4, 128), (10, 2, 64), (8, 1, 128)])
    case = {"op": op, "heads": heads, "kv": kv, "hd": hd}
    if op == "packed":
        case["type"] = rng.choice(["f32", "f32", "f16", "bf16"])
        case["seqs"] = _log_int(rng, 1, 24)
        # a padded square of scores no larger than the largest listed prompt's
        most = int(math.sqrt((4096 if case["type"] == "f32" else 8192) ** 2 * 32 * 128 / (case["seqs"] * heads * hd)))
        case["len"] = _log_int(rng, 1, min(most, 8192))
        return case
    case["type"], case["cache"] = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
    case["page"] = rng.choice([8, 16, 16, 20, 32, 64, 100, 256])
    case["seqs"] = _log_int(rng, 1, 64)
    if op == "append":
        case["len"] = _log_int(rng, 1, 8192 // case["seqs"] if case["seqs"] < 8 else 1024)
        case["rows"] = rng.choice([1, rng.randint(2, 9), case["len"]])
        case["rows"] = min(case["rows"], case["len"])
        return case
    bytes_a_position = case["seqs"] * kv * hd * 2 * SIZE[case["cache"]]
    case["len"] = _log_int(rng, 1, min(16000, 48 * 8000 * 8 * 128 * 2 * 2 // bytes_a_position))
    case["rows"] = min(case["len"], rng.choice([1, 1, 1, rng.randint(2, 9)]))
    return case


def _lens(case):
    """Positions of each sequence, the new rows among them: the longest first, then ragged ones."""
    rng = random.Random(case["seqs"] * 1000003 + case["len"])
    return [case["len"]] + [min(case["len"], _log_int(rng, max(1, case["len"] / 5), case["len"])) for _ in range(case["seqs"] - 1)]


def _rows(case):
    """New rows of each sequence: all (a prompt), one (decode), or up to case['rows'] (a verify step)."""
    lens = _lens(case)
    if case["op"] == "packed" or case["rows"] == case["len"]:
        return lens
    if case["rows"] == 1:
        return [1] * len(lens)
    rng = random.Random(case["rows"] * 7919 + case["seqs"])
    return [min(n, case["rows"]) if i == 0 else min(n, rng.randint(1, case["rows"])) for i, n in enumerate(lens)]


def _starts(rows):
    at = [0]
    for n in rows:
        at.append(at[-1] + n)
    return at


# ---------------------------------------------------------------- what a program has in hand
def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _angles(positions, hd):
    """(sin, cos) of every position and pair, [positions][hd / 2][2], from 64-bit angles."""
    rate = BASE ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * rate
    return torch.stack([torch.sin(angle), torch.cos(angle)], -1).float()


def _fused(case, rows, g):
    """One buffer of q, k, v rows as a fused projection leaves them, and its three views."""
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    x = torch.randn(rows, (h + 2 * kv) * hd, device="cuda", generator=g)
    # a few strong channels in the keys and queries, as trained models have them
    gain = torch.exp(0.4 * torch.randn(hd, device="cuda", generator=g))
    x[:, :(h + kv) * hd] *= gain.repeat(h + kv)
    x = x.to(TYPES[case["type"]])
    return x[:, :h * hd].view(rows, h, hd), x[:, h * hd:(h + kv) * hd].view(rows, kv, hd), x[:, (h + kv) * hd:].view(rows, kv, hd)


def _pages(case, g):
    """The pools, and each sequence's pages in them in shuffled order; a table a little wider than needed."""
    page, lens = case["page"], _lens(case)
    need = [-(-n // page) for n in lens]
    total, width = sum(need) + 3, max(need) + 2
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    for s, (at, n) in enumerate(zip(_starts(need), need)):
        table[s, :n] = order[at:at + n]
    shape = (total, page, case["kv"], case["hd"])
    gain = torch.exp(0.4 * torch.randn(case["hd"], device="cuda", generator=g))
    k = (torch.randn(shape, device="cuda", generator=g) * gain).to(TYPES[case["cache"]])
    v = torch.randn(shape, device="cuda", generator=g).to(TYPES[case["cache"]])
    return k, v, table


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens, rows = _lens(case), _rows(case)
    state = {"case": case, "longest": max(rows), "start": _ints(_starts(rows))}
    q, k, v = _fused(case, sum(rows), g)
    if case["op"] == "packed":
        return {**state, "q": q, "k": k, "v": v}
    state["k_pages"], state["v_pages"], state["table"] = _pages(case, g)
    state["lens"] = _ints(lens)
    # where each new row stands: its sequence and its position in it
    state["seq"] = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows)).cuda()
    if own:
        import nanocamelid_amd as nc
        state["cache"] = nc.PagedKV(state["k_pages"], state["v_pages"])
        state["batch"] = nc.PagedBatch(state["table"], state["lens"], None if case["rows"] == 1 else state["start"])
    if case["op"] == "append":
        return {**state, "q": q, "k": k, "v": v, "angles": _angles(case["len"], case["hd"])}
    return {**state, "q": q}


_CONTEXT = []


def _context():
    if not _CONTEXT:
        import nanocamelid_amd as nc
        _CONTEXT.append(nc.Context(torch.cuda.current_device()))
    return _CONTEXT[0]


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        import nanocamelid_amd as nc
        if op == "append":
            q, k = nc.paged_kv_append(_context(), state["cache"], state["batch"], state["k"], state["v"], state["angles"], q=state["q"], want_k=True)
            return {"q": q, "k": k, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}
        if op == "paged":
            return nc.paged_attention(_context(), state["cache"], state["batch"], state["q"])
        return nc.packed_attention(_context(), state["q"], state["k"], state["v"], state["start"])
    return {"append": _plain_append, "paged": _plain_paged, "packed": _plain_packed}[op](state)


def _positions(state):
    """Position of every new row in its sequence."""
    seq, start = state["seq"], state["start"]
    row = torch.arange(seq.numel(), device="cuda") - start[seq]
    return state["lens"][seq] - (start[seq + 1] - start[seq]) + row


def _turn(x, angles):
    sin, cos = angles[:, None, :, 0], angles[:, None, :, 1]
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _plain_append(state):
    page = state["case"]["page"]
    at = _positions(state)
    angles = state["angles"][at]
    q, k = _turn(state["q"], angles), _turn(state["k"], angles)
    where = state["table"][state["seq"], at // page]
    state["k_pages"][where, at % page] = k.to(state["k_pages"].dtype)
    state["v_pages"][where, at % page] = state["v"].to(state["v_pages"].dtype)
    return {"q": q.to(state["q"].dtype), "k": k.to(state["k"].dtype), "k_pages": state["k_pages"], "v_pages": state["v_pages"]}


def _padded(x, seq, row, seqs, longest):
    """Packed rows [T][heads][hd] as a padded float32 batch [seqs][heads][longest][hd]."""
    out = torch.zeros(seqs, longest, *x.shape[1:], device="cuda")
    out[seq, row] = x.float()
    return out.transpose(1, 2).contiguous()


def _softmax_product(q, k, v, seen, scale):
    """q [S][kv][group][n][hd], k and v [S][kv][m][hd], seen [S][n][m]: attention in float32, a row without keys zero."""
    s, kv, group, n, hd = q.shape
    score = (q.reshape(s, kv, group * n, hd) @ k.transpose(-1, -2).contiguous()).view(s, kv, group, n, -1) * scale
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = (weight.view(s, kv, group * n, -1) @ v).view(s, kv, group, n, hd)
    return torch.where(total > 0, out / total, 0.0)


def _plain_paged(state):
    case = state["case"]
    seqs, n, kv, hd = case["seqs"], state["longest"], case["kv"], case["hd"]
    table, start, seq = state["table"], state["start"], state["seq"]
    # every sequence's keys and values in order, padded to the table's width
    k = state["k_pages"][table].flatten(1, 2).float().transpose(1, 2).contiguous()
    v = state["v_pages"][table].flatten(1, 2).float().transpose(1, 2).contiguous()
    at = _positions(state)
    row = torch.arange(seq.numel(), device="cuda") - start[seq]
    q = _padded(state["q"], seq, row, seqs, n).view(seqs, kv, case["heads"] // kv, n, hd)
    last = torch.full((seqs, n), -1, dtype=at.dtype, device="cuda")
    last[seq, row] = at
    m = torch.arange(k.shape[2], device="cuda")
    # what lies behind a sequence's last position is not part of it
    v = v.masked_fill((m[None, :] >= state["lens"][:, None])[:, None, :, None], 0.0)
    out = _softmax_product(q, k, v, m[None, None, :] <= last[:, :, None], 1 / math.sqrt(hd))
    return out.flatten(1, 2)[seq, :, row].to(state["q"].dtype)


def _plain_packed(state):
    case = state["case"]
    seqs, n, kv, hd = case["seqs"], state["longest"], case["kv"], case["hd"]
    start = state["start"].long()
    t = torch.arange(state["q"].shape[0], device="cuda")
    seq = torch.searchsorted(start, t, right=True) - 1
    row = t - start[seq]
    q = _padded(state["q"], seq, row, seqs, n).view(seqs, kv, case["heads"] // kv, n, hd)
    k, v = _padded(state["k"], seq, row, seqs, n), _padded(state["v"], seq, row, seqs, n)
    m = torch.arange(n, device="cuda")
    seen = (m[None, :] <= m[:, None])[None].expand(seqs, n, n)
    out = _softmax_product(q, k, v, seen, 1 / math.sqrt(hd))
    return out.flatten(1, 2)[seq, :, row].to(state["q"].dtype)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    lens, rows = _lens(case), _rows(case)
    total, size = sum(rows), SIZE[case["type"]]
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(rows, lens))
    if case["op"] == "packed":
        return {"bytes": total * (2 * h + 2 * kv) * hd * size, "flops": 4 * pairs * h * hd}
    index = 4 * (sum(-(-m // case["page"]) for m in lens) + 2 * len(lens))
    if case["op"] == "append":
        angles = min(total, case["len"]) * hd * 4
        return {"bytes": total * hd * ((2 * h + 3 * kv) * size + 2 * kv * SIZE[case["cache"]]) + angles + 4 * total + 8 * len(lens), "flops": 3 * total * (h + kv) * hd}
    return {"bytes": 2 * sum(lens) * kv * hd * SIZE[case["cache"]] + 2 * total * h * hd * size + index, "flops": 4 * pairs * h * hd}


# ---------------------------------------------------------------- the results in 64 bits
def _turned(x, first, hd, angles):
    """Rows of one sequence, the first at position `first`, as complex pairs times e^(i angle)."""
    z = torch.view_as_complex(x.double().unflatten(-1, (hd // 2, 2)).contiguous())
    a = angles[first:first + x.shape[0]].double()
    return torch.view_as_real(z * torch.complex(a[..., 1].contiguous(), a[..., 0].contiguous())[:, None]).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    hd, group = case["hd"], case["heads"] // case["kv"]
    lens, rows = _lens(case), _rows(case)
    starts = _starts(rows)
    table = state["table"].tolist() if "table" in state else None
    if case["op"] == "append":
        page = case["page"]
        q = torch.cat([_turned(state["q"][a:a + n], m - n, hd, state["angles"]) for a, n, m in zip(starts, rows, lens)])
        k = torch.cat([_turned(state["k"][a:a + n], m - n, hd, state["angles"]) for a, n, m in zip(starts, rows, lens)])
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        at = torch.tensor([table[s][p // page] * page + p % page for s, (n, m) in enumerate(zip(rows, lens)) for p in range(m - n, m)]).cuda()
        k_pages.flatten(0, 1).index_copy_(0, at, k)
        v_pages.flatten(0, 1).index_copy_(0, at, state["v"].double())
        return {"q": q, "k": k, "k_pages": k_pages, "v_pages": v_pages}
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    for s, (a, n, m) in enumerate(zip(starts, rows, lens)):
        if table is None:
            keys, values = state["k"][a:a + m], state["v"][a:a + m]
        else:
            pages = state["table"][s, :-(-m // case["page"])].long()
            keys, values = (state[x][pages].flatten(0, 1)[:m] for x in ("k_pages", "v_pages"))
        hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        for h in range(case["heads"]):
            score = state["q"][a:a + n, h].double() @ keys[:, h // group].double().T / math.sqrt(hd)
            out[a:a + n, h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ values[:, h // group].double()
    return out
