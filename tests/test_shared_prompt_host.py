"""What the operators for continuations of one prompt refuse, and the plan of the shared attention: all of it without a GPU."""
import pytest
import torch

from imparo_b200.kernels import lib, ops


def test_tensors_off_the_device_are_refused():
    f, i = torch.ones(2), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ops.KernelError):
        ops.sample_filtered(torch.zeros(2, 9), f, f, i)
    with pytest.raises(ops.KernelError):
        ops.step_tables(i, i, i, i.view(2, 1), 16, 4, i.view(2, 1), i, i, i, i.long(), i, i)
    plan = ops.shared_prefix_plan(2, 1, 4, 2, 64, torch.bfloat16, 100, 10, sms=148)
    with pytest.raises(ops.KernelError):
        ops.paged_attention_shared(torch.zeros(2, 256), f, f, i, i, i.view(2, 1), 16, 4, i, i[:1], None, 1.0, f, f, f, plan, 4, 2, 64, i)


def test_entry_points_refuse_sizes_before_they_launch():
    k = lib.kernels()
    some = 1 << 20                                                 # a pointer that is never followed
    assert k.imparo_sample_filtered(some, 0, 10, some, some, None, None, None, some, None, 0, 10, None) == 0
    assert k.imparo_sample_filtered(some, 0, 10, None, some, None, None, None, some, None, 2, 10, None) == -7
    assert k.imparo_sample_filtered(some, 0, 10, some, None, None, None, None, some, None, 2, 10, None) == -7
    assert k.imparo_sample_filtered(some, 0, 10, some, some, None, None, None, some, None, 2, 0, None) == -2
    assert k.imparo_sample_filtered(some, 0, 9, some, some, None, None, None, some, None, 2, 10, None) == -2
    assert k.imparo_sample_filtered(some, 0, 1 << 25, some, some, None, None, None, some, None, 2, (1 << 24) + 1, None) == -2
    assert k.imparo_sample_filtered(some, 2, 10, some, some, None, None, None, some, None, 2, 10, None) == -1
    tables = lambda **kw: k.imparo_step_tables(*{**dict(l=some, c=some, f=some, nf=3, h=some, hw=2, p=None, s=None, n=2, ps=16, np=9, t=some, w=3,
                                                        pos=some, it=some, nt=5, rs=some, sl=some, tk=some, st=some, stream=None), **kw}.values())
    for bad in (dict(n=0), dict(ps=0), dict(np=0), dict(w=0), dict(hw=-1), dict(nf=-1), dict(nt=-1), dict(p=some)):
        assert tables(**bad) == -2, bad
    names = ("q", "qs", "k", "v", "dt", "pos", "it", "tab", "ni", "mb", "ps", "np", "gs", "sh", "ng", "win", "scale", "sinks", "out", "acc", "ml",
             "rows", "nh", "nkv", "hd", "cs", "ns", "co", "no", "st", "stream")
    base = dict(zip(names, (some, 256, some, some, 1, some, some, some, 2, 9, 16, 30, some, some, 1, 0, 1.0, None, some, some, some, 2, 4, 2, 64,
                            64, 2, 64, 1, some, None)))
    call = lambda **kw: k.imparo_attention_shared(*{**base, **kw}.values())
    assert call(rows=0) == 0
    for bad, code in ((dict(hd=8), -3), (dict(hd=72), -3), (dict(hd=272), -3), (dict(nkv=3), -5), (dict(nkv=0), -5), (dict(dt=3), -1),
                      (dict(ng=0), -2), (dict(ni=0), -2), (dict(mb=0), -2), (dict(ps=0), -2), (dict(np=0), -2), (dict(np=1 << 30), -2),
                      (dict(ns=0), -2), (dict(no=0), -2), (dict(cs=0), -2), (dict(co=0), -2), (dict(ns=2048), -2)):
        assert call(**bad) == code, bad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("rows,groups", [(1, 1), (8, 1), (64, 1), (256, 1), (132, 4), (64, 64), (4096, 7)])
@pytest.mark.parametrize("shared,own", [(0, 0), (0, 1), (1, 0), (100, 1), (2048, 300), (32768, 256), (100000, 5000), (1 << 20, 1 << 20), ((1 << 31) - 1, 5)])
def test_plans_cover_their_keys(rows, groups, shared, own, hd, dtype):
    for nh, nkv in ((32, 8), (8, 1), (4, 4)):
        p = ops.shared_prefix_plan(rows, groups, nh, nkv, hd, dtype, shared, own, sms=148)
        assert p.n_shared >= 1 and p.n_own >= 1 and p.n_shared + p.n_own <= ops.MAX_SPLITS
        assert p.n_shared * p.chunk_shared >= shared and p.n_own * p.chunk_own >= own
        assert p.acc_floats == rows * nh * (p.n_shared + p.n_own) * hd and p.ml_floats == 2 * rows * nh * (p.n_shared + p.n_own)


def test_plan_refusals():
    for args in ((0, 1, 4, 2, 64, torch.float32, 1, 1), (1, 0, 4, 2, 64, torch.float32, 1, 1), (1, 1, 4, 3, 64, torch.float32, 1, 1),
                 (1, 1, 4, 2, 64, torch.float32, -1, 1), (1, 1, 4, 2, 64, torch.float32, 1, -1)):
        with pytest.raises(ops.KernelError):
            ops.shared_prefix_plan(*args, sms=148)


def test_every_status_code_has_a_text():
    """The codes of csrc/kernels/common.cuh; what read_status says names the cause, not the code."""
    import os
    import re
    header = os.path.join(os.path.dirname(ops.__file__), "..", "csrc", "kernels", "common.cuh")
    with open(header) as f:
        codes = {name: int(code) for name, code in re.findall(r"#define IMPARO_ST_(\w+) (\d+)", f.read())}
    assert codes["STEP_SIZE"] == 5
    for code in codes.values():
        status = torch.tensor([code, 63, 2, -1], dtype=torch.int32)
        with pytest.raises(ops.KernelError, match=r"device check failed: [a-z][^0-9]{8,}\(kernel 63, index 2, value -1\)"):
            ops.read_status(status)
        assert not status.any()
