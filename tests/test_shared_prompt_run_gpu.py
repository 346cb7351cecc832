"""The operators together, as a program uses them that draws several continuations of each of its prompts, and the filters through
Engine.generate and the command line."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from imparo_b200.kernels import ops
from imparo_b200.sampling import Sampler, uniform_for
from tests.gpu_helpers import make_requests, model_dir
from tests.test_attention_shared_gpu import Batch
from tests.test_sample_filtered_gpu import plain_pick

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("graph", [False, True])
def test_several_continuations_of_two_prompts(dtype, graph):
    """Prompts of 83 and 40 positions, 5 and 3 continuations forked from them, 6 steps: tables, cache rows by slot, attention, pick."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    nh, nkv, hd, page, vocab, steps = 8, 2, 64, 16, 501, 6
    prompts, each = [83, 40], [5, 3]
    rows, n_pages, width = sum(each), 60, 12
    draw = lambda *shape, scale=1.0: torch.randn(*shape, device=DEV, generator=gen) * scale
    embed, w_q, w_kv, w_out = draw(vocab, 96), draw(96, nh * hd, scale=0.15), draw(96, 2 * nkv * hd, scale=0.1), draw(nh * hd, vocab, scale=0.3)
    k, v = (torch.full((n_pages, page, nkv * hd), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=DEV)
    status = ops.new_status(DEV)

    def tables(lengths, counts, held, free, parent=None, shared=None):
        n, total = len(lengths), int(sum(counts))
        outs = [torch.empty(n, width, dtype=torch.int32, device=DEV), i32(np.zeros(total)), i32(np.zeros(total)), i32(np.zeros(n + 1)),
                torch.zeros(total, dtype=torch.int64, device=DEV), i32([0])]
        ops.step_tables(i32(lengths), i32(counts), i32(free), held, page, n_pages, *outs, status, parent=parent, shared=shared)
        ops.read_status(status)
        return outs

    free = list(range(n_pages))
    # the prompts' own step
    held, positions, items, _, slots, taken = tables([0, 0], prompts, i32(np.full((2, width), -1)), free)
    free = free[int(taken):]
    k.view(-1, nkv * hd)[slots], v.view(-1, nkv * hd)[slots] = (x.to(dtype) for x in draw(sum(prompts), 2 * nkv * hd).split(nkv * hd, dim=1))
    # the fork: continuations hold nothing yet but their parent's whole pages; the rest of the prompt is copied into their own page
    of = [g for g, n in enumerate(each) for _ in range(n)]
    everyone = torch.cat([held, i32(np.full((rows, width), -1))])
    parent, shared = i32([-1, -1] + of), i32([0, 0] + [prompts[g] // page * page for g in of])
    lengths = [prompts[0], prompts[1]] + [prompts[g] // page * page for g in of]
    counts = [0, 0] + [prompts[g] % page for g in of]
    table, _, _, start, slots, taken = tables(lengths, counts, everyone, free, parent, shared)
    free = free[int(taken):]
    for r, g in enumerate(of):
        mine = slots[int(start[2 + r]):int(start[3 + r])]
        where = held[g, prompts[g] // page].long() * page + torch.arange(len(mine), device=DEV)
        for x in (k, v):
            x.view(-1, nkv * hd)[mine] = x.view(-1, nkv * hd)[where]
    held, lengths = table[2:].contiguous(), [prompts[g] for g in of]
    assert all(torch.equal(held[r, :prompts[g] // page], table[g, :prompts[g] // page]) for r, g in enumerate(of))

    group_start, shared_len = i32([0, 5, 8]), i32([prompts[0] // page * page, prompts[1] // page * page])
    plan = ops.shared_prefix_plan(rows, 2, nh, nkv, hd, dtype, 80, 30)
    acc, ml = torch.empty(plan.acc_floats, device=DEV), torch.empty(plan.ml_floats, device=DEV)
    q, out = (torch.zeros(rows, nh * hd, dtype=dtype, device=DEV) for _ in range(2))
    table, positions, items, start, slots, taken = (torch.empty_like(held), i32(np.zeros(rows)), i32(np.zeros(rows)), i32(np.zeros(rows + 1)),
                                                    torch.zeros(rows, dtype=torch.int64, device=DEV), i32([0]))
    lens, ones, free_dev = i32(lengths), i32(np.ones(rows)), i32(np.resize(free, 30))
    temps, us = torch.full((rows,), 0.9, device=DEV), torch.zeros(rows, device=DEV)
    top_k, top_p, min_p = i32([0, 40, 0, 300, 7, 0, 90, 1]), torch.tensor([0.9, 1.0, 0.5, 0.95, 1.0, 1.0, 0.8, 1.0], device=DEV), torch.full((rows,), 0.01, device=DEV)
    tokens, kept, logits = i32(np.arange(rows) * 31 % vocab), i32(np.zeros(rows)), torch.zeros(rows, vocab, device=DEV)

    def step():
        ops.step_tables(lens, ones, free_dev, held, page, n_pages, table, positions, items, start, slots, taken, status)
        x = embed[tokens.long()]
        rows_kv = (x @ w_kv).to(dtype)
        q.copy_(x @ w_q)
        k.view(-1, nkv * hd)[slots], v.view(-1, nkv * hd)[slots] = rows_kv[:, :nkv * hd], rows_kv[:, nkv * hd:]
        ops.paged_attention_shared(q, k, v, positions, items, table, page, n_pages, group_start, shared_len, None, hd ** -0.5, out, acc, ml, plan,
                                   nh, nkv, hd, status)
        logits.copy_(out.float() @ w_out)
        ops.sample_filtered(logits, temps, us, tokens, top_k=top_k, top_p=top_p, min_p=min_p, kept=kept)

    captured = None
    for n in range(steps):
        us.copy_(torch.tensor([uniform_for(100 + r, n) for r in range(rows)]))
        if graph and n > 0:
            if captured is None:
                torch.cuda.synchronize()
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured):
                    step()
            captured.replay()
        else:
            step()
        ops.read_status(status)
        assert positions.tolist() == lengths and items.tolist() == list(range(rows))
        b = Batch.__new__(Batch)
        b.nh, b.nkv, b.hd, b.page, b.dtype, b.scale = nh, nkv, hd, page, dtype, hd ** -0.5
        b.q, b.k, b.v, b.table, b.positions, b.items = q, k, v, table, positions, items
        want, bound = b.plain()
        assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
        x = logits.double().cpu().numpy()
        assert list(zip(tokens.tolist(), kept.tolist())) == [
            plain_pick(x[r], np.float32(0.9), np.float32(us[r].item()), int(top_k[r]), np.float32(top_p[r].item()), np.float32(0.01)) for r in range(rows)]
        used = int(taken)
        free = free[used:]
        free_dev.copy_(i32(np.resize(free, 30)))
        held.copy_(table)
        lengths = [length + 1 for length in lengths]
        lens.add_(1)
    assert len(free) < 60 - 9                                      # pages were taken on the way


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_a_padded_step_is_captured_once(dtype, hd):
    """Eight continuations of two prompts, of which others rest or have ended in every step: tables, cache rows and attention, with nothing
    between them, in one graph for eight rows.  The rows behind the step's tokens change nothing; the others are as in a step of their number."""
    nh, nkv, page, n_pages, width, rows = 8, 2, 16, 100, 12, 8
    rng = np.random.default_rng(hd)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(hd)
    i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=DEV)
    new = lambda n: i32(np.zeros(n))
    prompts, of = [80, 32], [0, 0, 0, 0, 0, 1, 1, 1]
    free = list(range(n_pages))                                    # (page 0 is the first prompt's first)
    whole = [[free.pop(0) for _ in range(n // page)] for n in prompts]
    held = np.full((rows, width), -1)
    for r, g in enumerate(of):
        held[r, :len(whole[g])] = whole[g]
    lengths = np.array([prompts[g] for g in of])
    draw = lambda *shape: torch.randn(*shape, device=DEV, generator=gen).to(dtype)
    k = torch.cat([torch.full((1, page, nkv * hd), 5.0, device=DEV, dtype=dtype), draw(n_pages, page, nkv * hd)])        # a page before the arena
    v = k.flip(0).contiguous()
    k_plain, v_plain = k.clone(), v.clone()
    inv_freq = 10000.0 ** (-torch.arange(hd // 2, device=DEV, dtype=torch.float32) / (hd // 2))
    plan = ops.shared_prefix_plan(rows, 2, nh, nkv, hd, dtype, 80, 30)
    acc, ml, status = torch.empty(plan.acc_floats, device=DEV), torch.empty(plan.ml_floats, device=DEV), ops.new_status(DEV)
    qkv, q, out = draw(rows, (nh + 2 * nkv) * hd), torch.zeros(rows, nh * hd, dtype=dtype, device=DEV), torch.zeros(rows, nh * hd, dtype=dtype, device=DEV)

    def reads(qkv, q, k, v, positions, items, table, group_start, shared, out):
        ops.qk_norm_rope_store(qkv, positions, items, None, None, inv_freq, hd, 1e-6, q, k[1:], v[1:], table, page, n_pages, nh, nkv, hd, status)
        ops.paged_attention_shared(q, k[1:], v[1:], positions, items, table, page, n_pages, group_start, shared, None, hd ** -0.5, out, acc, ml,
                                   plan, nh, nkv, hd, status)

    lens, counts, free_dev, held_dev, shared = i32(lengths), new(rows), new(rows), i32(held), i32(prompts)
    table, positions, items, start, slots, taken = torch.empty_like(held_dev), new(rows), new(rows), new(rows + 1), torch.zeros(rows, dtype=torch.int64, device=DEV), new(1)
    group_start = i32([0, 5, 8])

    def step():
        ops.step_tables(lens, counts, free_dev, held_dev, page, n_pages, table, positions, items, start, slots, taken, status)
        reads(qkv, q, k, v, positions, items, table, group_start, shared, out)

    def replay():
        nonlocal graph
        if graph is None:
            step()                                                 # (kernels configure themselves at their first launch)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        graph.replay()

    graph = None
    for n in range(8):
        active = np.array([1] * 8 if n == 0 else [0] * 8 if n == 7 else rng.integers(0, 2, 8))
        if n == 5:
            active[:5] = 0                                         # the first group rests
        for dst, src in ((lens, lengths), (counts, active), (free_dev, free[:rows]), (held_dev, held),
                         (group_start, [0, active[:5].sum(), active.sum()])):
            dst.copy_(i32(src))
        qkv.copy_(draw(*qkv.shape))
        replay()
        ops.read_status(status)
        t = int(active.sum())
        who = np.flatnonzero(active)
        for r in who:
            if held[r, lengths[r] // page] < 0:
                held[r, lengths[r] // page] = free.pop(0)
        assert positions.tolist() == lengths[who].tolist() + [-1] * (rows - t)
        if t:
            q_plain, out_plain = torch.zeros(t, nh * hd, dtype=dtype, device=DEV), torch.zeros(t, nh * hd, dtype=dtype, device=DEV)
            reads(qkv[:t], q_plain, k_plain, v_plain, i32(lengths[who]), i32(who), i32(held), group_start, shared, out_plain)
            assert torch.equal(out[:t], out_plain) and out_plain.any()
        assert not out[t:].any() and torch.equal(k, k_plain) and torch.equal(v, v_plain)
        lengths[who] += 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_streams_at_once(dtype):
    """Two programs' steps side by side on one device, each with buffers of its own: as one after the other."""
    batches = [Batch([(20, 700), (3, 100)], lambda r: 1 + 5 * r, 8, 2, 64, dtype, seed=s) for s in (1, 2)]
    rng = np.random.default_rng(1)
    logits = [torch.tensor(rng.standard_normal((5, 30000)) * 2, dtype=torch.float32, device=DEV) for _ in range(2)]
    ones, half = torch.ones(5, device=DEV), torch.full((5,), 0.5, device=DEV)
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)
    plan = ops.shared_prefix_plan(23, 2, 8, 2, 64, dtype, 700, 120)
    programs = []
    for b, x in zip(batches, logits):
        table, positions, items = torch.empty_like(b.table), i32(23), i32(23)
        scratch = [torch.empty(plan.acc_floats, device=DEV), torch.empty(plan.ml_floats, device=DEV)]
        made = [table, positions, items, i32(24), torch.zeros(23, dtype=torch.int64, device=DEV), i32(1)]
        lens, counts, free, out, ids = b.positions.clone(), i32(23) + 1, i32(1), torch.empty_like(b.q), i32(5)

        def step(b=b, x=x, made=made, scratch=scratch, lens=lens, counts=counts, free=free, out=out, ids=ids):
            ops.step_tables(lens, counts, free, b.table, b.page, b.n_pages, *made, b.status)
            ops.paged_attention_shared(b.q, b.k, b.v, made[1], made[2], made[0], b.page, b.n_pages, b.group_start, b.shared, None, b.scale, out,
                                       *scratch, plan, 8, 2, 64, b.status)
            ops.sample_filtered(x, ones, half, ids, top_p=half)
        programs.append((step, out, ids, b))
    want = []
    for step, out, ids, _ in programs:
        step()
        torch.cuda.synchronize()
        want.append((out.clone(), ids.clone()))
        out.zero_()
        ids.zero_()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (step, *_rest) in zip(streams, programs):
            with torch.cuda.stream(stream):
                step()
    torch.cuda.synchronize()
    for (_, out, ids, b), (w_out, w_ids) in zip(programs, want):
        ops.read_status(b.status)
        assert torch.equal(out, w_out) and torch.equal(ids, w_ids)


def test_sampler_rows_with_and_without_filters():
    """A row without a filter is picked as it always was, whatever its neighbours ask for."""
    rng = np.random.default_rng(4)
    logits = torch.tensor(rng.standard_normal((9, 5000)) * 2, dtype=torch.float32, device=DEV)
    sampler = Sampler(DEV, 4)
    temps, seeds, steps = [0.0, 0.7, 1.0, 1.2, 0.8, 0.9, 1.0, 0.0, 1.0], list(range(9)), [3] * 9
    top_ks, top_ps, min_ps = [5, 0, 50, 0, 0, 30, 0, 0, 1 << 40], [1.0, 1.0, 1.0, 0.8, 1.0, 0.9, 1.0, 0.5, 1.0], [0, 0, 0, 0, 0.05, 0.01, 0, 0, 0]
    plain = sampler.sample(logits, temps, seeds, steps)
    got = sampler.sample(logits, temps, seeds, steps, top_ks, top_ps, min_ps)
    x = logits.double().cpu().numpy()
    for r in range(9):
        if temps[r] == 0 or (top_ks[r] == 0 and top_ps[r] == 1 and min_ps[r] == 0):
            assert got[r] == plain[r]
        else:
            assert got[r] == plain_pick(x[r], np.float32(temps[r]), np.float32(uniform_for(r, 3)), min(top_ks[r], 1 << 30), np.float32(top_ps[r]),
                                        np.float32(min_ps[r]))[0]
    everyone = sampler.sample(logits[1:2], [0.7], [1], [3], [0], [0.6], [0])
    assert everyone[0] == plain_pick(x[1], np.float32(0.7), np.float32(uniform_for(1, 3)), 0, np.float32(0.6), 0)[0]
    assert sampler.sample(logits, temps, seeds, steps, [0] * 9, [1.0] * 9, None) == plain


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generate_with_filters(dtype):
    """Greedy, plain and filtered requests in one batch; what a request gets is what it gets alone, and every filtered pick is among the
    tokens its filters leave of the logits that the engine gives for the same tokens."""
    from imparo_b200.engine import Engine, StepItem
    prompts = list(make_requests("B", [5, 23, 40, 11], seed=1).values())
    kw = dict(temperature=[0.0, 0.8, 0.8, 1.1], seed=[0, 11, 12, 13], top_k=[0, 0, 20, 0], top_p=[1.0, 1.0, 0.9, 0.7], min_p=[0.0, 0.0, 0.02, 0.0])
    eng = Engine(model_dir("B"), dtype=dtype, ctx=64, parallel=4, page_size=4, num_pages=64, max_step_tokens=16)
    got = eng.generate(prompts, max_tokens=10, stop_token_ids=[], **kw)
    plain = eng.generate(prompts, max_tokens=10, stop_token_ids=[], temperature=kw["temperature"], seed=kw["seed"])
    assert got[0] == plain[0] and got[1] == plain[1] and (got[2] != plain[2] or got[3] != plain[3])
    for i in (2, 3):
        eng.add_request(900 + i)
        for at in range(0, len(prompts[i]), 16):                   # portions of the step's budget
            part = list(prompts[i])[at:at + 16]
            logits = eng.step([StepItem(900 + i, part, [len(part) - 1])])
        for n, token in enumerate(got[i]):
            row = logits[0].double()
            top = row.max()
            weight = torch.exp((row - top) / kw["temperature"][i])
            order = torch.argsort(row, descending=True)
            # (a little wider than the filters: the same tokens in another step's shape give logits a rounding apart)
            stay = order[:kw["top_k"][i] + 2] if kw["top_k"][i] else order
            w = weight[stay]
            stay = stay[((w.cumsum(0) - w) < (kw["top_p"][i] + 0.02) * w.sum()) & (w > 0.8 * kw["min_p"][i])]
            assert token in stay.tolist()
            logits = eng.step([StepItem(900 + i, [token], [0])])
        eng.end_request(900 + i)


def test_generate_refuses_bad_filters():
    from imparo_b200.engine import Engine
    eng = Engine(model_dir("A"), dtype="float32", ctx=64, parallel=2, page_size=16, num_pages=4)
    for kw in (dict(top_k=-1), dict(top_k=1.5), dict(top_p=0.0), dict(top_p=1.1), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=2.0),
               dict(top_k=[1, 2])):
        with pytest.raises(ValueError):
            eng.generate([[1, 2, 3]], max_tokens=2, temperature=1.0, **kw)


def test_command_line_filters():
    args = [sys.executable, "-m", "imparo_b200", "-m", model_dir("A"), "--decode", "6", "--json", "--dtype", "float32", "-c", "64", "--temperature", "1.0"]
    run = lambda *more: json.loads(subprocess.run(args + list(more) + ["1", "2", "3"], cwd=ROOT, capture_output=True, text=True, check=True).stdout)["tokens"][0]
    greedy = json.loads(subprocess.run(args[:-2] + ["1", "2", "3"], cwd=ROOT, capture_output=True, text=True, check=True).stdout)["tokens"][0]
    assert run("--top-k", "1") == greedy == run("--top-p", "0.000001") == run("--min-p", "1.0")
    assert run("--top-k", "50", "--top-p", "0.9", "--min-p", "0.01") == run("--top-k", "50", "--top-p", "0.9", "--min-p", "0.01")
