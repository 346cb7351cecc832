"""What the operators for several continuations of one prompt are measured on: picking tokens under filters, attention of rows that
share a prefix, and the block tables of a step made on the device.

Kinds:

  sample      one token per row of logits, from given random numbers, at a temperature and under top-k, top-p and min-p
  attention   one-token rows over the paged cache; the rows of a group share the pages of their first positions
  tables      the step's block tables, positions and slot map from the requests' lengths, new pages from the list of free ones

`run` computes them in plain torch operations, or, where `own` is true, by the calls a user makes of `imparo_b200.kernels.ops`.
"""
import math

import numpy as np
import torch

own = False

F32, BF16 = "float32", "bfloat16"
_DTYPE = {F32: torch.float32, BF16: torch.bfloat16}


def listed():
    return [
        # a single user's chat with the usual settings: latency
        {"name": "sample_1x65536_k40_p95", "kind": "sample", "rows": 1, "vocab": 65536, "dtype": F32, "mode": "chat"},
        # a small server, nucleus sampling alone: the sum goes over the whole vocabulary
        {"name": "sample_8x65536_p90", "kind": "sample", "rows": 8, "vocab": 65536, "dtype": F32, "mode": "nucleus"},
        # a busy server with a ragged vocabulary and 16-bit logits, every request with settings of its own
        {"name": "sample_61x32003_bf16_mixed", "kind": "sample", "rows": 61, "vocab": 32003, "dtype": BF16, "mode": "mixed"},
        # the largest batch over a large vocabulary
        {"name": "sample_256x131072_mixed", "kind": "sample", "rows": 256, "vocab": 131072, "dtype": F32, "mode": "mixed"},
        # eight continuations of one prompt: the benchmark's model, prompt and page size
        {"name": "attention_8_of_2048", "kind": "attention", "dtype": BF16, "groups": 1, "rows": 8, "shared": 2048, "own": 100, "heads": 32,
         "kv_heads": 8, "dim": 64, "page": 16},
        # the 32-bit path, which results are checked with: a few rows, an odd prompt
        {"name": "attention_f32_5_of_1001", "kind": "attention", "dtype": F32, "groups": 1, "rows": 5, "shared": 1001, "own": 33, "heads": 16,
         "kv_heads": 8, "dim": 64, "page": 16},
        # a system prompt before four long documents, each with many questions, wide heads
        {"name": "attention_4x33_of_8000_d128", "kind": "attention", "dtype": BF16, "groups": 4, "rows": 33, "shared": 8000, "own": 150,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32},
        # a busy server, every request behind one long document
        {"name": "attention_64_of_32768", "kind": "attention", "dtype": BF16, "groups": 1, "rows": 64, "shared": 32768, "own": 256, "heads": 32,
         "kv_heads": 8, "dim": 64, "page": 16},
        # the largest: a whole batch of continuations of a very long document
        {"name": "attention_256_of_100000", "kind": "attention", "dtype": BF16, "groups": 1, "rows": 256, "shared": 100000, "own": 200,
         "heads": 32, "kv_heads": 8, "dim": 64, "page": 16},
        # a decode step of a small server
        {"name": "tables_8_decode", "kind": "tables", "items": 8, "held": 2048, "tokens": 1, "page": 16, "forked": False},
        # 256 continuations forked from long prompts in one step
        {"name": "tables_256_forked", "kind": "tables", "items": 256, "held": 32768, "tokens": 1, "page": 16, "forked": True},
        # a large step of prompt portions
        {"name": "tables_500_portions", "kind": "tables", "items": 500, "held": 20000, "tokens": 200, "page": 16, "forked": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["sample", "sample", "attention", "attention", "attention", "tables"])
    if kind == "sample":
        return {"kind": kind, "rows": _log(rng, 1, 256), "vocab": _log(rng, 1000, 131072), "dtype": rng.choice([F32, F32, BF16]),
                "mode": rng.choice(["chat", "nucleus", "mixed"])}
    if kind == "tables":
        return {"kind": kind, "items": _log(rng, 1, 500), "held": _log(rng, 1, 32768), "tokens": _log(rng, 1, 100),
                "page": rng.choice([16, 16, 32, 64, 128]), "forked": rng.choice([False, True])}
    if rng.random() < 0.2:
        return {"kind": kind, "dtype": F32, "groups": rng.randint(1, 3), "rows": rng.randint(1, 12), "shared": _log(rng, 20, 4000),
                "own": _log(rng, 1, 300), "heads": 16, "kv_heads": rng.choice([4, 8]), "dim": 64, "page": 16}
    dim = rng.choice([64, 64, 128])
    return {"kind": kind, "dtype": BF16, "groups": rng.randint(1, 4), "rows": _log(rng, 1, 48), "shared": _log(rng, 100, 40000 * 64 // dim),
            "own": _log(rng, 1, 400), "heads": rng.choice([16, 24, 32]), "kv_heads": 8, "dim": dim, "page": rng.choice([16, 32, 64])}


# ---- inputs -------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    state = {"case": case}
    if case["kind"] == "sample":
        _prepare_sample(case, state, gen, rng)
    elif case["kind"] == "attention":
        _prepare_attention(case, state, gen, rng)
    else:
        _prepare_tables(case, state, rng)
    return state


def _prepare_sample(case, state, gen, rng):
    n, vocab = case["rows"], case["vocab"]
    # a model's logits: a broad bell, a few likely continuations well above it, some tokens forbidden
    logits = torch.randn(n, vocab, device="cuda", generator=gen) * 2.5
    likely = torch.randint(0, vocab, (n, 12), device="cuda", generator=gen)
    logits.scatter_add_(1, likely, torch.rand(n, 12, device="cuda", generator=gen) * 8.0)
    forbidden = torch.randint(0, vocab, (n, 5), device="cuda", generator=gen)
    logits.scatter_(1, forbidden, float("-inf"))
    state["logits"] = logits.to(_DTYPE[case["dtype"]])
    temperature = rng.uniform(0.6, 1.3, n)
    top_k, top_p, min_p = np.zeros(n, dtype=np.int32), np.ones(n), np.zeros(n)
    if case["mode"] == "chat":
        top_k[:], top_p[:] = 40, 0.95
    elif case["mode"] == "nucleus":
        top_p[:] = rng.uniform(0.85, 0.97, n)
    else:                                   # every row its own: greedy, plain, each filter alone and all together
        which = rng.integers(0, 6, n)
        temperature[which == 0] = 0.0
        some_k = np.exp(rng.uniform(np.log(1), np.log(vocab), n)).astype(np.int32)
        top_k[(which == 2) | (which == 5)] = some_k[(which == 2) | (which == 5)]
        top_p[(which == 3) | (which == 5)] = rng.uniform(0.3, 0.99, n)[(which == 3) | (which == 5)]
        min_p[(which == 4) | (which == 5)] = np.exp(rng.uniform(np.log(1e-4), np.log(0.3), n))[(which == 4) | (which == 5)]
    uniform = rng.integers(0, 1 << 24, n) / float(1 << 24)
    for name, values in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p), ("uniform", uniform)):
        state[name] = torch.tensor(values, dtype=torch.float32, device="cuda")
    state["top_k"] = torch.tensor(top_k, dtype=torch.int32, device="cuda")
    state["ids"] = torch.empty(n, dtype=torch.int32, device="cuda")
    state["kept"] = torch.empty(n, dtype=torch.int32, device="cuda")


def _attention_sizes(case):
    """Per group its shared positions, per row its own ones (the lengths differ, as in a batch that has run for a while)."""
    rng = np.random.default_rng(case["rows"] * 131 + case["shared"])
    groups, rows = case["groups"], case["rows"]
    shared = [max(1, case["shared"] - int(case["shared"] * 0.3 * g / groups)) for g in range(groups)]
    own_positions = [int(rng.integers(max(1, case["own"] // 2), case["own"] + 1)) for _ in range(groups * rows)]
    return shared, own_positions


def _prepare_attention(case, state, gen, rng):
    page, width = case["page"], case["kv_heads"] * case["dim"]
    shared, own_positions = _attention_sizes(case)
    rows = case["groups"] * case["rows"]
    # a group's whole pages are shared; the page in which its shared positions end is a row's own from there on, so a row
    # that goes on in it has a copy of it
    n_blocks = [-(-(shared[r // case["rows"]] + own_positions[r]) // page) for r in range(rows)]
    whole = [s // page for s in shared]
    n_pages = sum(whole) + sum(n_blocks[r] - whole[r // case["rows"]] for r in range(rows)) + 3
    pages = rng.permutation(n_pages).astype(np.int32)
    table = np.full((rows, max(n_blocks) + 2), -1, dtype=np.int32)
    at = 0
    copies = []
    for g in range(case["groups"]):
        first = pages[at:at + whole[g]]
        at += whole[g]
        for r in range(g * case["rows"], (g + 1) * case["rows"]):
            mine = n_blocks[r] - whole[g]
            table[r, :whole[g]] = first
            table[r, whole[g]:n_blocks[r]] = pages[at:at + mine]
            at += mine
            if shared[g] % page and r > g * case["rows"]:
                copies.append((table[g * case["rows"], whole[g]], table[r, whole[g]], shared[g] % page))
    dtype = _DTYPE[case["dtype"]]
    k = torch.randn(n_pages, page, width, device="cuda", generator=gen).to(dtype)
    v = torch.randn(n_pages, page, width, device="cuda", generator=gen).to(dtype)
    for src, dst, filled in copies:
        k[int(dst), :filled] = k[int(src), :filled]
        v[int(dst), :filled] = v[int(src), :filled]
    # queries twice as long as the keys' scale: a softmax with some weight on few keys
    q = (torch.randn(rows, case["heads"] * case["dim"], device="cuda", generator=gen) * 2.0).to(dtype)
    to_device = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")
    state.update(k=k, v=v, q=q, table=to_device(table), n_pages=n_pages,
                 positions=to_device([shared[r // case["rows"]] + own_positions[r] - 1 for r in range(rows)]),
                 items=to_device(list(range(rows))), group_start=to_device([g * case["rows"] for g in range(case["groups"] + 1)]),
                 shared=to_device(shared), most_shared=max(shared), most_own=max(own_positions), out=torch.empty_like(q),
                 scale=1.0 / math.sqrt(case["dim"]))
    if own:
        from imparo_b200.kernels import ops
        state["status"] = ops.new_status("cuda")
        state["plan"] = plan = ops.shared_prefix_plan(rows, case["groups"], case["heads"], case["kv_heads"], case["dim"], dtype,
                                                      most_shared=max(shared), most_own=max(own_positions))
        state["part_acc"] = torch.empty(plan.acc_floats, dtype=torch.float32, device="cuda")
        state["part_ml"] = torch.empty(plan.ml_floats, dtype=torch.float32, device="cuda")


def _counts(case):
    """The new tokens of every item."""
    if case["tokens"] == 1:
        return np.ones(case["items"], dtype=np.int64)
    return np.random.default_rng(case["items"] * 131 + case["tokens"]).integers(1, 2 * case["tokens"], case["items"])


def _prepare_tables(case, state, rng):
    items, page = case["items"], case["page"]
    lengths = rng.integers(max(0, case["held"] // 2), case["held"] + 1, items)
    counts = _counts(case)
    parent, shared = np.full(items, -1), np.zeros(items, dtype=np.int64)
    if case["forked"]:                       # every eighth item is a prompt, the seven behind it go on from its whole pages
        for r in range(items):
            if r % 8:
                parent[r] = r - r % 8
                shared[r] = lengths[r] = lengths[r - r % 8] // page * page
    mapped = np.where(parent < 0, -(-lengths // page), 0)
    blocks = -(-(lengths + counts) // page)
    need = int((blocks - np.where(parent < 0, mapped, shared // page)).sum())
    n_pages = int(mapped.sum()) + need + 7
    pages = rng.permutation(n_pages).astype(np.int32)
    width = -(-(case["held"] + 2 * case["tokens"]) // page)
    held = np.full((items, width), -1, dtype=np.int32)
    at = 0
    for r in range(items):
        held[r, :mapped[r]] = pages[at:at + mapped[r]]
        at += mapped[r]
    free = np.sort(pages[at:])               # the lowest free page is handed out first
    total = int(counts.sum())
    to_device = lambda values: torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")
    state.update(lengths=to_device(lengths), counts=to_device(counts), free=to_device(free), held=to_device(held), n_pages=n_pages,
                 total=total, parent=to_device(parent) if case["forked"] else None, shared=to_device(shared) if case["forked"] else None,
                 table=torch.empty_like(to_device(held)), positions=to_device(np.zeros(total)), items=to_device(np.zeros(total)),
                 row_start=to_device(np.zeros(items + 1)), slots=torch.empty(total, dtype=torch.int64, device="cuda"),
                 taken=to_device([0]))
    if own:
        from imparo_b200.kernels import ops
        state["status"] = ops.new_status("cuda")


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"sample": _own_sample, "attention": _own_attention, "tables": _own_tables}[kind](state)
    return {"sample": _plain_sample, "attention": _plain_attention, "tables": _plain_tables}[kind](state)


def _own_sample(s):
    from imparo_b200.kernels import ops
    ops.sample_filtered(s["logits"], s["temperature"], s["uniform"], s["ids"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                        kept=s["kept"])
    return s["ids"], s["kept"]


def _own_attention(s):
    from imparo_b200.kernels import ops
    c = s["case"]
    ops.paged_attention_shared(s["q"], s["k"], s["v"], s["positions"], s["items"], s["table"], c["page"], s["n_pages"], s["group_start"],
                               s["shared"], None, s["scale"], s["out"], s["part_acc"], s["part_ml"], s["plan"], c["heads"],
                               c["kv_heads"], c["dim"], s["status"])
    return s["out"]


def _own_tables(s):
    from imparo_b200.kernels import ops
    ops.step_tables(s["lengths"], s["counts"], s["free"], s["held"], s["case"]["page"], s["n_pages"], s["table"], s["positions"], s["items"],
                    s["row_start"], s["slots"], s["taken"], s["status"], parent=s["parent"], shared=s["shared"])
    return s["table"], s["positions"], s["items"], s["row_start"], s["slots"], s["taken"]


def _plain_sample(s):
    # 64 bits: what is kept and picked depends on running sums next to a border
    v = s["logits"].double()
    n, vocab = v.shape
    v = torch.where(torch.isnan(v), float("-inf"), v)
    order = torch.sort(v, dim=1, descending=True, stable=True)
    top = order.values[:, :1]
    temperature = s["temperature"].double()[:, None]
    safe = torch.where(temperature > 0, temperature, 1.0)
    weight = torch.where(order.values == top, 1.0, torch.exp((order.values - top) / safe))
    live = order.values > float("-inf")
    rank = torch.arange(vocab, device=v.device)[None]
    top_k = s["top_k"].long()[:, None]
    keep = live & ((top_k <= 0) | (rank < top_k))
    weight = weight * keep
    before = weight.cumsum(1) - weight
    top_p = s["top_p"].double()[:, None]
    keep &= (top_p >= 1) | (before < top_p * weight.sum(1, keepdim=True)) | (rank == 0)
    keep &= (weight >= s["min_p"].double()[:, None]) | (rank == 0)
    keep &= (temperature > 0) | (rank == 0)
    in_order = torch.zeros_like(v).scatter_(1, order.indices, weight * keep)
    sums = in_order.cumsum(1)
    past = sums > s["uniform"].double()[:, None] * sums[:, -1:]
    ids = past.int().argmax(1)
    return ids.int(), keep.sum(1).int()


def _gather(cache, table, positions, page):
    """Rows of the cache at positions [n] of one table row, in 32 bits."""
    return cache[table[positions // page].long(), positions % page].float()


def _plain_attention(s):
    c = s["case"]
    heads, kv_heads, dim, page, per = c["heads"], c["kv_heads"], c["dim"], c["page"], c["rows"]
    each = heads // kv_heads
    rows = c["groups"] * per
    q = s["q"].float().view(rows, kv_heads, each, dim)
    out = torch.empty(rows, kv_heads, each, dim, device=q.device)
    shared, own_positions = _attention_sizes(c)
    for g in range(c["groups"]):
        r0, r1 = g * per, (g + 1) * per
        most = max(own_positions[r0:r1])
        k0, v0 = (_gather(x, s["table"][r0], torch.arange(shared[g], device=q.device), page).view(-1, kv_heads, dim) for x in (s["k"], s["v"]))
        # the rows' own positions, side by side; those behind a row's last one are masked
        at = shared[g] + torch.arange(most, device=q.device)
        seen = at[None] <= s["positions"][r0:r1, None]
        blocks = torch.clamp(at // page, max=s["table"].shape[1] - 1)
        pages = torch.where(seen, s["table"][r0:r1][:, blocks], 0).long()
        k1, v1 = (x[pages, (at % page)[None]].float().view(per, most, kv_heads, dim) for x in (s["k"], s["v"]))
        for h in range(kv_heads):
            qh = q[r0:r1, h]
            a = (qh.reshape(-1, dim) @ k0[:, h].t()).view(per, each, -1) * s["scale"]
            b = (qh @ k1[:, :, h].transpose(1, 2)) * s["scale"]
            b = torch.where(seen[:, None], b, float("-inf"))
            top = torch.maximum(a.amax(2), b.amax(2))[..., None]
            a, b = torch.exp(a - top), torch.exp(b - top)
            total = a.sum(2) + b.sum(2)
            o = (a.view(-1, shared[g]) @ v0[:, h]).view(per, each, dim) + b @ torch.where(seen[:, :, None], v1[:, :, h], 0.0)
            out[r0:r1, h] = o / total[..., None]
    return out.view(rows, heads * dim).to(s["q"].dtype)


def _plain_tables(s):
    page = s["case"]["page"]
    lengths, counts, held = s["lengths"].long(), s["counts"].long(), s["held"]
    items, width = held.shape
    device = held.device
    block = torch.arange(width, device=device)[None]
    table = held
    if s["parent"] is not None:
        from_parent = held[torch.clamp(s["parent"], min=0).long()]
        table = torch.where((s["parent"] >= 0)[:, None] & (block < (s["shared"].long() // page)[:, None]), from_parent, held)
    wanted = (block >= (lengths // page)[:, None]) & (block * page < (lengths + counts)[:, None]) & (counts > 0)[:, None]
    new = wanted & (table < 0)
    number = (new.flatten().cumsum(0) - 1).view(items, width)
    taken = new.sum()
    table = torch.where(new, s["free"][torch.clamp(number, 0, s["free"].numel() - 1)], table)
    row_start = torch.cat([torch.zeros(1, dtype=torch.long, device=device), counts.cumsum(0)])
    token = torch.arange(s["total"], device=device)
    item = torch.searchsorted(row_start[1:], token, right=True)
    position = lengths[item] + token - row_start[item]
    slot = table[item, position // page].long() * page + position % page
    return table, position.int(), item.int(), row_start.int(), slot, taken.int().view(1)


# ---- what a pass cannot do without, and its result in 64 bits ---------------------------------------------------------------

def work(case):
    if case["kind"] == "sample":
        n, vocab = case["rows"], case["vocab"]
        return {"bytes": n * vocab * (4 if case["dtype"] == F32 else 2) + n * 28, "flops": n * vocab * 4}
    if case["kind"] == "attention":
        shared, own_positions = _attention_sizes(case)
        size = 4 if case["dtype"] == F32 else 2
        rows = case["groups"] * case["rows"]
        keys = sum(shared) + sum(own_positions)
        seen = sum(shared) * case["rows"] + sum(own_positions)
        blocks = sum(s // case["page"] for s in shared) + sum(-(-o // case["page"]) for o in own_positions)
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size + 2 * rows * case["heads"] * case["dim"] * size + 4 * blocks,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    items, tokens = case["items"], int(_counts(case).sum())
    width = -(-(case["held"] + 2 * case["tokens"]) // case["page"])
    new = -(-tokens // case["page"])
    # a held entry that is mapped is read, every entry of the table is written
    read = items * (case["held"] * 3 // 4) // case["page"]
    return {"bytes": 4 * (read + items * width + new + 5 * items) + 16 * tokens, "flops": 0}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(state)
    if case["kind"] == "attention":
        return _exact_attention(state)
    return None                              # whole numbers


def _exact_sample(s):
    logits = s["logits"].double().cpu().numpy()
    column = lambda name: s[name].cpu().numpy()
    temperature, top_k, top_p, min_p, uniform = (column(x) for x in ("temperature", "top_k", "top_p", "min_p", "uniform"))
    ids, kept = [], []
    for r in range(logits.shape[0]):
        numbers = np.flatnonzero(logits[r] > -np.inf)
        if numbers.size == 0:
            ids.append(0), kept.append(0)
            continue
        x = logits[r][numbers]
        top = x.max()
        if not temperature[r] > 0:
            ids.append(int(numbers[x.argmax()])), kept.append(1)
            continue
        falling = np.lexsort((numbers, -x))
        if top_k[r] > 0:
            falling = falling[:top_k[r]]
        w = np.exp((x[falling] - top) / np.float64(temperature[r])).astype(np.longdouble)
        if top_p[r] < 1:
            before = np.concatenate([[np.longdouble(0)], np.cumsum(w)[:-1]])
            enough = max(1, int((before < np.longdouble(top_p[r]) * w.sum()).sum()))
            falling, w = falling[:enough], w[:enough]
        enough = max(1, int((w >= np.longdouble(min_p[r])).sum()))
        falling, w = falling[:enough], w[:enough]
        rising = np.sort(falling)
        sums = np.cumsum(np.exp((x[rising] - top) / np.float64(temperature[r])).astype(np.longdouble))
        ids.append(int(numbers[rising[np.searchsorted(sums, np.longdouble(uniform[r]) * sums[-1], side="right")]]))
        kept.append(len(rising))
    return torch.tensor(ids, dtype=torch.int32), torch.tensor(kept, dtype=torch.int32)


def _exact_attention(s):
    """Row by row over all of its positions, in 64 bits."""
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for r in range(s["q"].shape[0]):
        at = torch.arange(int(s["positions"][r]) + 1, device=out.device)
        flat = s["table"][r].long()[at // page] * page + at % page
        k, v = (x.view(-1, kv_heads, dim)[flat].double().permute(1, 0, 2) for x in (s["k"], s["v"]))
        scores = torch.bmm(s["q"][r].double().view(kv_heads, heads // kv_heads, dim), k.transpose(1, 2)) * s["scale"]
        out[r] = torch.bmm(torch.softmax(scores, dim=2), v).reshape(-1)
    return out
