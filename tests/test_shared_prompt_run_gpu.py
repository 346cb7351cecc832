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
