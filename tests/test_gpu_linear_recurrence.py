"""Gated linear recurrences on the GPU against the row-by-row float64 definition, within the bounds that the
roundings of the arithmetic allow (sequence_oracle)."""
import itertools

import numpy as np
import pytest
import torch

import pysiglib_b200 as psl
import sequence_oracle as so
from pysiglib_b200 import load_cusig, torch_api

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16


def make(seed, batch, rows, dim, gates, dtype, gate_dtype, form, initial, sequences=0, dense_offsets=True):
    g = torch.Generator().manual_seed(seed)
    lead = () if sequences else (batch,)
    x = torch.randn(*lead, rows, dim, generator=g, dtype=F64).to(dtype)
    logits = 2.0 + 1.5 * torch.randn(*lead, rows, gates, generator=g, dtype=F64)
    gate = {"value": torch.sigmoid(logits) * torch.where(torch.rand(logits.shape, generator=g) < 0.1, -1.0, 1.0).double(),
            "log": torch.nn.functional.logsigmoid(logits), "logit": logits}[form].to(gate_dtype)
    derivs = torch.randn(*lead, rows, dim, generator=g, dtype=F64).to(dtype)
    count = sequences or batch
    wide = so.state_type(dtype)
    start = torch.randn(count, dim, generator=g, dtype=F64).to(wide) if initial else None
    tail = torch.randn(count, dim, generator=g, dtype=F64).to(wide)
    offsets = None
    if sequences:
        lo, hi = (0, rows) if dense_offsets else (min(3, rows), max(min(3, rows), rows - 5))
        cuts = torch.randint(lo, hi + 1, (sequences - 1,), generator=g).sort().values
        offsets = torch.cat([torch.tensor([lo]), cuts, torch.tensor([hi])])
    return x, gate, start, derivs, tail, offsets


def cuda(t):
    return None if t is None else t.cuda()


def run_and_check(data, form, complement, checkpoints=True, tail=True, **kw):
    x, gate, start, derivs, state_derivs, offsets = data
    state_derivs = state_derivs if tail else None
    expect = so.recurrence(x, gate, start, form, complement, offsets, derivs, state_derivs)
    how = {"gate_form": form, "complement": complement, "offsets": cuda(offsets)}
    X, G, S = cuda(x), cuda(gate), cuda(start)
    before = load_cusig.launch_count()
    h, state, marks = psl.linear_recurrence(X, G, S, return_state=True, return_checkpoints=True, **how)
    dx, dgate, dinitial = psl.linear_recurrence_backprop(cuda(derivs), X, G, S, state_derivs=cuda(state_derivs),
                                                         checkpoints=marks if checkpoints else None, **how)
    assert load_cusig.launch_count() > before
    assert h.dtype == x.dtype and dgate.dtype == gate.dtype and state.dtype == so.state_type(x.dtype)
    for name, got in (("h", h), ("state", state), ("dx", dx), ("dgate", dgate)):
        so.check(got, expect[name], name)
    if start is None:
        assert dinitial is None
    else:
        so.check(dinitial, expect["dinitial"], "dinitial")
    return h


TYPES = [(F32, F32), (F64, F64), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]


@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 31, 33, 63, 64, 65, 127, 129, 200, 513, 1030])
@pytest.mark.parametrize("dim", [1, 3, 4, 17, 32, 100])
def test_sizes(rows, dim):
    form = ("value", "log", "logit")[rows % 3]
    run_and_check(make(rows * 7 + dim, 2, rows, dim, dim, F32, F32, form, rows % 2 == 0), form, rows % 4 > 1)


@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("form", ["value", "log", "logit"])
@pytest.mark.parametrize("complement", [False, True])
def test_types_and_forms(dtype, gate_dtype, form, complement):
    for dim in (24, 21):
        run_and_check(make(dim, 3, 150, dim, dim, dtype, gate_dtype, form, True), form, complement)


@pytest.mark.parametrize("dim,gates", [(64, 1), (64, 2), (64, 16), (96, 2), (40, 8), (340, 85), (34, 17), (15, 3), (51, 3),
                                       (384, 3), (1024, 4), (260, 1)])
@pytest.mark.parametrize("dtype,gate_dtype", [(F32, F32), (F64, F64), (BF16, F32), (F16, F16)])
def test_shared_gates(dim, gates, dtype, gate_dtype):
    run_and_check(make(dim + gates, 2, 75, dim, gates, dtype, gate_dtype, "logit", True), "logit", gates % 2 == 0)


@pytest.mark.parametrize("rows,sequences", [(1, 1), (1, 5), (6, 9), (40, 3), (64, 64), (150, 7), (300, 1), (515, 40), (1300, 300), (900, 700)])
@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("dtype,gate_dtype,dim", [(F32, F32, 36), (BF16, F32, 35), (F64, F64, 6)])
def test_packed_sequences(rows, sequences, dense, dtype, gate_dtype, dim):
    data = make(rows + sequences, 1, rows, dim, dim, dtype, gate_dtype, "log", rows % 2 == 0, sequences, dense)
    h = run_and_check(data, "log", rows % 3 == 0)
    offsets = data[-1]
    outside = torch.ones(rows, dtype=torch.bool)
    outside[int(offsets[0]):int(offsets[-1])] = False
    assert (h.cpu()[outside] == 0).all()


def test_packed_is_each_sequence_alone():
    x, gate, start, derivs, tail, offsets = make(3, 1, 400, 20, 5, F32, F32, "logit", True, 11)
    how = {"gate_form": "logit", "complement": True}
    packed, state = psl.linear_recurrence(cuda(x), cuda(gate), cuda(start), offsets=offsets.to(torch.int32), return_state=True, **how)
    expect = so.recurrence(x, gate, start, "logit", True, offsets)
    for k, (lo, hi) in enumerate(so.spans_of(offsets, 400)):
        h, s = psl.linear_recurrence(cuda(x)[lo:hi], cuda(gate)[lo:hi], cuda(start)[k], return_state=True, **how)
        so.check(h, (packed[lo:hi].cpu().double(), 2 * expect["h"][1][lo:hi]), "h")
        so.check(s, (state[k].cpu().double(), 2 * expect["state"][1][k]), "state")


@pytest.mark.parametrize("checkpoints,tail,initial", list(itertools.product([True, False], repeat=3)))
def test_backward_with_and_without_its_optional_parts(checkpoints, tail, initial):
    run_and_check(make(5, 2, 333, 48, 48, BF16, F32, "log", initial), "log", False, checkpoints, tail)
    run_and_check(make(6, 1, 333, 10, 5, F32, F32, "value", initial, 9, False), "value", True, checkpoints, tail)


def test_many_channels_and_long_rows():
    run_and_check(make(1, 3, 70, 1999, 1999, F32, F32, "logit", True), "logit", True)
    run_and_check(make(2, 70, 20, 260, 260, BF16, BF16, "log", True), "log", False)
    run_and_check(make(3, 1, 20000, 8, 8, F32, F32, "log", True), "log", True)
    run_and_check(make(4, 1, 9000, 12, 3, BF16, F32, "logit", False, 13), "logit", False)
    run_and_check(make(5, 2, 5000, 1, 1, F64, F64, "value", True), "value", False)


def test_views_are_read_in_place():
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(2, 3, 90, 4 * 24, generator=g)
    x, gate, derivs = wide[..., :24], wide[..., 24:48], wide[..., 48:72]
    expect = so.recurrence(x.reshape(6, 90, 24), gate.reshape(6, 90, 24), None, "logit", True, None, derivs.reshape(6, 90, 24))
    W = wide.cuda()
    X, G, D = W[..., :24], W[..., 24:48], W[..., 48:72]
    h, marks = psl.linear_recurrence(X, G, gate_form="logit", complement=True, return_checkpoints=True)
    dx, dgate, _ = psl.linear_recurrence_backprop(D, X, G, gate_form="logit", complement=True, checkpoints=marks)
    for name, got in (("h", h), ("dx", dx), ("dgate", dgate)):
        so.check(got.reshape(6, 90, 24), expect[name], name)
    # rows and batch swapped, an odd start, channels apart, a gate for all rows and batch entries
    for view in (lambda t: t.transpose(0, 1), lambda t: t[:, 1:, 3:20], lambda t: t[..., ::2], lambda t: t[:, ::3]):
        base = torch.randn(40, 41, 24, generator=g)
        v = view(base)
        one = torch.randn(1, 1, v.shape[-1], generator=g).expand(*v.shape)
        expect = so.recurrence(v.contiguous(), one.contiguous(), None, "logit", False, None, v.contiguous())
        V, O = view(base.cuda()), one[:1, :1].contiguous().cuda().expand(*v.shape)
        so.check(psl.linear_recurrence(V, O, gate_form="logit"), expect["h"], "h")
        dx, dgate, _ = psl.linear_recurrence_backprop(V, V, O, gate_form="logit")
        so.check(dx, expect["dx"], "dx")
        so.check(dgate, expect["dgate"], "dgate")


def test_a_sequence_keeps_its_nan_and_infinities_to_itself():
    x, gate, start, derivs, tail, offsets = make(9, 1, 700, 33, 33, F32, F32, "log", True, 6)
    offsets = torch.tensor([0, 5, 130, 131, 300, 600, 700])
    expect = so.recurrence(x, gate, start, "log", False, offsets, derivs, tail)
    bad = x.clone()
    bad_gate = gate.clone()
    bad[200], bad[400], bad_gate[130], derivs_bad = float("nan"), float("inf"), float("nan"), derivs.clone()
    derivs_bad[200] = float("nan")
    how = {"gate_form": "log", "offsets": cuda(offsets)}
    h, state = psl.linear_recurrence(cuda(bad), cuda(bad_gate), cuda(start), return_state=True, **how)
    dx, dgate, dinitial = psl.linear_recurrence_backprop(cuda(derivs_bad), cuda(bad), cuda(bad_gate), cuda(start), state_derivs=cuda(tail), **how)
    clean = [0, 1, 5]
    for k in clean:
        lo, hi = int(offsets[k]), int(offsets[k + 1])
        for name, got in (("h", h), ("dx", dx), ("dgate", dgate)):
            so.check(got[lo:hi], (expect[name][0][lo:hi], expect[name][1][lo:hi]), "%s of %d" % (name, k))
        so.check(state[k], (expect["state"][0][k], expect["state"][1][k]), "state")
        so.check(dinitial[k], (expect["dinitial"][0][k], expect["dinitial"][1][k]), "dinitial")
    assert torch.isnan(h[200:300]).all() and not torch.isfinite(h[400:600]).any() and torch.isnan(h[130]).all()


@pytest.mark.parametrize("form,closed,open_", [("value", 0.0, 1.0), ("log", -float("inf"), 0.0), ("logit", -float("inf"), float("inf"))])
def test_gates_that_are_closed_or_open(form, closed, open_):
    x = torch.randn(2, 300, 20, generator=torch.Generator().manual_seed(2))
    gate = torch.full((2, 300, 20), open_)
    gate[:, ::50] = closed
    so.check(psl.linear_recurrence(x.cuda(), gate.cuda(), gate_form=form), so.recurrence(x, gate, None, form, False)["h"], "h")
    h = psl.linear_recurrence(x.cuda(), gate.cuda(), gate_form=form, complement=True)
    so.check(h, so.recurrence(x, gate, None, form, True)["h"], "h")
    lowest = torch.full((2, 300, 20), torch.finfo(F32).min if form != "value" else 0.0)
    h = psl.linear_recurrence(x.cuda(), lowest.cuda(), gate_form=form, complement=True)
    assert torch.equal(h.cpu(), x)


@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("dim,gates", [(32, 32), (32, 4), (7, 7), (9, 3)])
def test_steps_continue_a_prompt(dtype, gate_dtype, dim, gates):
    x, gate, start, *_ = make(11, 3, 40, dim, gates, dtype, gate_dtype, "logit", True)
    for complement in (False, True):
        expect = so.recurrence(x, gate, start, "logit", complement)
        X, G = cuda(x), cuda(gate)
        _, state = psl.linear_recurrence(X[:, :25], G[:, :25], cuda(start), gate_form="logit", complement=complement, return_state=True)
        for t in range(25, 40):
            out = psl.linear_recurrence_step(X[:, t], G[:, t], state, gate_form="logit", complement=complement)
            so.check(out, (expect["h"][0][:, t], expect["h"][1][:, t]), "row %d" % t)
        so.check(state, expect["state"], "state")


def test_gradients_against_differences():
    x, gate, start, derivs, tail, offsets = (t.cuda() if t is not None else None for t in make(21, 1, 12, 6, 2, F64, F64, "logit", True, 3))
    for form, complement in itertools.product(("value", "log", "logit"), (False, True)):
        leaves = [t.clone().requires_grad_() for t in (x, gate if form != "log" else -gate.abs(), start)]

        def f(*args):
            return torch_api.linear_recurrence(*args, gate_form=form, complement=complement, offsets=offsets, return_state=True)
        assert torch.autograd.gradcheck(f, leaves, eps=1e-6, atol=1e-6, rtol=1e-5)


def test_autograd_partial_gradients():
    x, gate, start, derivs, tail, _ = make(22, 2, 70, 8, 8, F32, F32, "logit", True)
    expect = so.recurrence(x, gate, start, "logit", False, None, torch.zeros_like(derivs), tail)
    X, G, S = (t.cuda().requires_grad_() for t in (x, gate, start))
    h, state = torch_api.linear_recurrence(X, G, S, gate_form="logit", return_state=True)
    gx, gg, gs = torch.autograd.grad(state, (X, G, S), tail.cuda())
    for name, got in (("dx", gx), ("dgate", gg), ("dinitial", gs)):
        so.check(got, expect[name], name)
    only = torch_api.linear_recurrence(X, G.detach(), gate_form="logit")
    only.sum().backward()
    expect = so.recurrence(x, gate, None, "logit", False, None, torch.ones_like(derivs))
    so.check(X.grad, expect["dx"], "dx")
    assert G.grad is None


def test_same_bits_on_every_run():
    x, gate, start, derivs, tail, offsets = (cuda(t) for t in make(23, 1, 3000, 192, 3, BF16, F32, "log", True, 17))
    def once():
        h, marks = psl.linear_recurrence(x, gate, start, gate_form="log", offsets=offsets, return_checkpoints=True)
        return (h, *psl.linear_recurrence_backprop(derivs, x, gate, start, gate_form="log", offsets=offsets, checkpoints=marks))
    first = once()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_side_streams_and_graphs():
    sets = [make(30 + k, 2, 260, 96, 1, F32, F32, "logit", True) for k in range(2)]
    expects = [so.recurrence(x, gate, start, "logit", True, None, derivs) for x, gate, start, derivs, *_ in sets]
    static = [[cuda(t) for t in s[:4]] for s in sets]

    def both(x, gate, start, derivs):
        h, marks = psl.linear_recurrence(x, gate, start, gate_form="logit", complement=True, return_checkpoints=True)
        return (h, *psl.linear_recurrence_backprop(derivs, x, gate, start, gate_form="logit", complement=True, checkpoints=marks))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = []
    for k in range(2):
        with torch.cuda.stream(streams[k]):
            results.append(both(*static[k]))
    torch.cuda.synchronize()
    names = ("h", "dx", "dgate", "dinitial")
    for k in range(2):
        for name, got in zip(names, results[k]):
            so.check(got, expects[k][name], name)
    # two captured calls, replayed in turns and on other inputs
    graphs, outs = [], []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both(*static[k]))
        graphs.append(graph)
    for order in ((0, 1), (1, 0)):
        for k in order:
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            for name, got in zip(names, outs[k]):
                so.check(got, expects[k][name], name)
    for a, b in zip(static[0], static[1]):
        a.copy_(b)
    graphs[0].replay()
    torch.cuda.synchronize()
    for name, got in zip(names, outs[0]):
        so.check(got, expects[1][name], name)


def test_more_than_32_bits_of_elements():
    rows, dim = (1 << 31) // 1024 + 4096, 1024
    x = torch.zeros(rows, dim, dtype=BF16, device="cuda")
    gate = torch.full((1, 1), 0.5, dtype=BF16, device="cuda").expand(rows, 1)
    x[rows - 3] = 1.0
    h, state = psl.linear_recurrence(x, gate, return_state=True)
    assert float(h[: rows - 3].abs().max()) == 0
    assert h[rows - 3:, 7].tolist() == [1.0, 0.5, 0.25] and h[rows - 1].unique().numel() == 1
    assert float(state.min()) == float(state.max()) == 0.25


@pytest.mark.parametrize("dtype", [np.float32, np.float64, np.float16])
def test_host_arrays(dtype):
    t = {np.float32: F32, np.float64: F64, np.float16: F16}[dtype]
    x, gate, start, derivs, tail, offsets = make(40, 1, 90, 12, 4, t, t, "logit", True, 5)
    expect = so.recurrence(x, gate, start, "logit", True, offsets, derivs, tail)
    to = lambda v: v.numpy()
    how = {"gate_form": "logit", "complement": True, "offsets": to(offsets)}
    h, state, marks = psl.linear_recurrence(to(x), to(gate), to(start), return_state=True, return_checkpoints=True, **how)
    assert isinstance(h, np.ndarray) and h.dtype == dtype
    for m in (marks, None):
        dx, dgate, dinitial = psl.linear_recurrence_backprop(to(derivs), to(x), to(gate), to(start), state_derivs=to(tail), checkpoints=m, **how)
        for name, got in (("h", h), ("state", state), ("dx", dx), ("dgate", dgate), ("dinitial", dinitial)):
            so.check(torch.from_numpy(got), expect[name], name)
    cpu = psl.linear_recurrence(x.to(t), gate, start, gate_form="logit", complement=True, offsets=offsets)
    assert cpu.device.type == "cpu"
    so.check(cpu, expect["h"], "h")
    s = to(start).copy()
    out = psl.linear_recurrence_step(to(x)[:5], to(gate)[:5], s, gate_form="logit", complement=True)
    one = so.recurrence(x[:5, None], gate[:5, None], start, "logit", True)
    so.check(torch.from_numpy(out), (one["h"][0][:, 0], one["h"][1][:, 0]), "step")
    so.check(torch.from_numpy(s), one["state"], "state")


@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("rows,dim,gates,sequences", [(5000, 64, 64, 0), (3001, 33, 33, 0), (4100, 128, 2, 9), (2500, 20, 20, 40)])
def test_rows_cut_into_segments(dtype, gate_dtype, rows, dim, gates, sequences):
    """One batch entry, few channels: the rows are shared out over the SMs and joined."""
    form = "log" if sequences else "logit"
    run_and_check(make(rows + dim, 1, rows, dim, gates, dtype, gate_dtype, form, True, sequences), form, dim == 64, rows % 2 == 0)


@pytest.mark.parametrize("batch,rows,dim,dtype", [(80, 150, 128, F32), (64, 70, 1024, BF16), (700, 40, 64, F16), (3, 40, 8200, F32),
                                                  (2500, 9, 16, F64), (130, 33, 130, BF16)])
def test_many_strips(batch, rows, dim, dtype):
    run_and_check(make(batch, batch, rows, dim, dim, dtype, dtype, "logit", True), "logit", False)


@pytest.mark.parametrize("dim", [4, 12, 20, 36])
@pytest.mark.parametrize("dtype,gate_dtype", [(BF16, BF16), (F16, F32)])
def test_sixteen_bit_rows_aligned_to_eight_bytes(dim, dtype, gate_dtype):
    run_and_check(make(dim, 2, 100, dim, dim, dtype, gate_dtype, "logit", True), "logit", True)
    g = torch.Generator().manual_seed(dim)
    wide = torch.randn(2, 90, 64, generator=g).to(dtype)
    view = lambda t: t[..., 4:4 + dim]  # dense rows of 128 bytes that start 8 bytes in
    gate = torch.randn(2, 90, dim, generator=g).to(gate_dtype)
    expect = so.recurrence(view(wide).contiguous(), gate, None, "logit", False, None, view(wide).contiguous())
    W = wide.cuda()
    dx, dgate, _ = psl.linear_recurrence_backprop(view(W), view(W), gate.cuda(), gate_form="logit")
    so.check(psl.linear_recurrence(view(W), gate.cuda(), gate_form="logit"), expect["h"], "h")
    so.check(dx, expect["dx"], "dx")
    so.check(dgate, expect["dgate"], "dgate")


def test_a_captured_training_step():
    """Warmed up on a side stream, as torch asks for: a graph that was made eagerly on the default stream and still
    lives would tie the leaves to that stream, for any torch operation."""
    x, gate, start, derivs, tail, _ = make(50, 2, 300, 32, 4, F32, F32, "logit", True)
    expect = so.recurrence(x, gate, start, "logit", True, None, derivs, tail)
    X, G, S = (cuda(t).requires_grad_() for t in (x, gate, start))
    D, T = cuda(derivs), cuda(tail)

    def step():
        h, state = torch_api.linear_recurrence(X, G, S, gate_form="logit", complement=True, return_state=True)
        return torch.autograd.grad((h, state), (X, G, S), (D, T))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for name, got in zip(("dx", "dgate", "dinitial"), grads):
        so.check(got, expect[name], name)


def test_calls_from_two_threads():
    import threading
    sets = [make(60 + k, 1, 2000, 64, 2, BF16, F32, "log", True, 7) for k in range(2)]
    expects = [so.recurrence(*s[:3], "log", False, s[5], s[3]) for s in sets]
    failures = []

    def work(k):
        try:
            x, gate, start, derivs, _, offsets = (cuda(t) for t in sets[k])
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                for _ in range(20):
                    h = psl.linear_recurrence(x, gate, start, gate_form="log", offsets=offsets)
                    grads = psl.linear_recurrence_backprop(derivs, x, gate, start, gate_form="log", offsets=offsets)
            stream.synchronize()
            for name, got in zip(("h", "dx", "dgate", "dinitial"), (h, *grads)):
                so.check(got, expects[k][name], name)
        except BaseException as e:  # noqa: BLE001
            failures.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failures, failures


def test_the_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    code = ("import torch, pysiglib_b200 as psl\n"
            "x = torch.randn(2, 300, 48, device='cuda'); g = torch.randn(2, 300, 1, device='cuda')\n"
            "graph = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(graph):\n"
            "    h = psl.linear_recurrence(x, g, gate_form='logit')\n"
            "    d = psl.linear_recurrence_backprop(x, x, g, gate_form='logit')[1]\n"
            "graph.replay(); torch.cuda.synchronize()\n"
            "assert torch.equal(h, psl.linear_recurrence(x, g, gate_form='logit'))\n"
            "assert torch.equal(d, psl.linear_recurrence_backprop(x, x, g, gate_form='logit')[1])\n")
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_offsets_that_are_out_of_order_stay_in_bounds():
    """Device offsets are trusted; wrong ones give wrong numbers for their own sequences and nothing else: memory around
    the arrays stays as it was."""
    rows, dim = 200, 16
    whole = torch.full((3 * rows, dim), 7.0, device="cuda")
    x = whole[rows:2 * rows]
    gate = torch.full((rows, dim), 0.5, device="cuda")
    for bad in ([0, 150, 50, 200], [-5, 10, 300], [90, 80, 70, 60], [2 ** 40, -2 ** 40, 5], [200, 200, 200]):
        offsets = torch.tensor(bad, device="cuda")
        start = torch.zeros(len(bad) - 1, dim, device="cuda")
        psl.linear_recurrence(x, gate, start, offsets=offsets, return_state=True)
        psl.linear_recurrence_backprop(x, x, gate, start, offsets=offsets)
    torch.cuda.synchronize()
    assert (whole == 7.0).all()
    expect = so.recurrence(x.cpu()[None], gate.cpu()[None], None, "value", False)["h"]
    so.check(psl.linear_recurrence(x, gate), tuple(t[0] for t in expect), "h")


def test_what_a_graph_has_kept_is_not_overwritten_unseen():
    x, gate, start, derivs, _, _ = make(60, 1, 40, 8, 8, F32, F32, "logit", True)
    X = cuda(x[0]).requires_grad_()
    G, S = cuda(gate[0])[None], cuda(start)
    h = torch_api.linear_recurrence(X[None], G, S, gate_form="logit")
    psl.linear_recurrence_step(X[:1].detach(), G[0, :1], S, gate_form="logit")
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    # offsets on the host are the caller's again after the call
    offsets = np.array([0, 15, 40])
    h = torch_api.linear_recurrence(X, G[0], gate_form="logit", offsets=offsets)
    offsets[1] = 3
    (got,) = torch.autograd.grad(h, X, cuda(derivs[0]))
    expect = psl.linear_recurrence_backprop(cuda(derivs[0]), X.detach(), G[0], gate_form="logit", offsets=np.array([0, 15, 40]))[0]
    assert torch.equal(got, expect)


@pytest.mark.parametrize("lengths", [(900, 3, 0, 0, 1100, 997), (1, 2998, 1), (0, 3000, 0), (7,) * 400, (100, 2000)])
def test_segments_of_packed_rows_that_begin_and_end_in_sequences(lengths):
    """Sequence bounds before, in, at and behind the cuts between segments; rows before the first and behind the last."""
    rows = 3000
    x, gate, _, derivs, _, _ = make(61, 1, rows, 24, 24, F32, F32, "log", False)
    x, gate, derivs = x[0], gate[0], derivs[0]
    bounds = np.cumsum([0, *lengths])
    bounds = bounds + min(5, rows - bounds[-1])
    rng = np.random.default_rng(62)
    start, tail = (torch.from_numpy(rng.standard_normal((len(lengths), 24)).astype(np.float32)) for _ in range(2))
    run_and_check((x, gate, start, derivs, tail, torch.from_numpy(bounds)), "log", True)


@pytest.mark.parametrize("view", [lambda t: t[:, None, :3], lambda t: t[:, None, :1], lambda t: t[None, :, 1:4, None],
                                  lambda t: t[1:2, None, :1].expand(3, 7, 1, -1, -1), lambda t: t[:, None].transpose(0, 2)])
def test_views_with_axes_of_one_entry(view):
    """Three and more batch axes, some of one entry, as x, gate and derivatives."""
    g = torch.Generator().manual_seed(70)
    bases = [torch.randn(4, 5, 40, 12, generator=g) for _ in range(3)]
    X, G, D = (view(t.cuda()) for t in bases)
    batch = X.shape[:-2].numel()
    flat = [view(t).reshape(batch, 40, 12) for t in bases]
    expect = so.recurrence(flat[0], flat[1], None, "logit", True, None, flat[2])
    h, marks = psl.linear_recurrence(X, G, gate_form="logit", complement=True, return_checkpoints=True)
    dx, dgate, _ = psl.linear_recurrence_backprop(D, X, G, gate_form="logit", complement=True, checkpoints=marks)
    for name, got in (("h", h), ("dx", dx), ("dgate", dgate)):
        assert got.shape == X.shape
        so.check(got.reshape(batch, 40, 12), expect[name], name)


@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
def test_gates_far_below_zero(dtype, gate_dtype):
    """Logits whose gate is tiny or 0: a state as large as its type lets through what the gate says and no more, with
    `complement` and in the gradients too.  Smallest gate: 2^-100 of float32's range, 2^-1000 of float64's."""
    far = {F32: [-60.0, -66.0, -75.0, -80.0], F64: [-60.0, -600.0, -695.0, -700.0]}[so.state_type(dtype)] + [-float("inf")]
    dim = len(far) * 4
    gate = torch.tensor(far, dtype=F64).repeat_interleave(4).to(gate_dtype).expand(2, 3, dim).contiguous()
    x = torch.zeros(2, 3, dim, dtype=dtype)
    big = 1e30 if so.state_type(dtype) is F32 else 1e300
    start = torch.full((2, dim), big, dtype=so.state_type(dtype))
    closed = torch.isinf(gate[0, 0])
    for complement in (False, True):
        # -inf is exact below; the oracle's bound for 16-bit gates grows with the finite ones alone
        bound = so.recurrence(x[..., ~closed], gate[..., ~closed], start[:, ~closed], "logit", complement, None,
                              torch.ones_like(x[..., ~closed]))
        X, G, S = cuda(x), cuda(gate), cuda(start)
        h, state = psl.linear_recurrence(X, G, S, gate_form="logit", complement=complement, return_state=True)
        dx, dgate, dinitial = psl.linear_recurrence_backprop(torch.ones_like(X), X, G, S, gate_form="logit", complement=complement)
        for name, got in (("h", h), ("state", state), ("dx", dx), ("dgate", dgate), ("dinitial", dinitial)):
            so.check(got[..., ~closed], bound[name], name)
            assert (got[..., closed].cpu() == (1.0 if name == "dx" else 0.0)).all(), name
        step_state = S.clone()
        psl.linear_recurrence_step(X[:, 0], G[:, 0], step_state, gate_form="logit", complement=complement)
        so.check(step_state[:, ~closed], so.recurrence(x[:, :1, ~closed], gate[:, :1, ~closed], start[:, ~closed], "logit", complement)["state"], "step")
        assert (step_state[:, closed] == 0).all()


@pytest.mark.parametrize("rows", [40, 3000])
def test_a_first_gate_that_is_not_finite(rows):
    """a_0 times an absent state is a_0 times 0, NaN here, in a packed sequence as in a dense one; the next is clean."""
    x, gate, _, derivs, _, _ = make(71, 1, rows, 8, 8, F32, F32, "value", False)
    gate[0, 0, 0], gate[0, 0, 1] = float("nan"), float("inf")
    X, G, cut = cuda(x[0]), cuda(gate[0]), rows - 10
    dense, packed = psl.linear_recurrence(X, G), psl.linear_recurrence(X, G, offsets=torch.tensor([0, cut, rows]))
    assert torch.isnan(dense[:, :2]).all() and torch.isnan(packed[:cut, :2]).all()
    expect = so.recurrence(x[0], gate[0].clamp(-1, 1).nan_to_num(0.0), None, "value", False, torch.tensor([0, cut, rows]))["h"]
    so.check(packed[:, 2:], tuple(t[:, 2:] for t in expect), "h")
    so.check(packed[cut:], tuple(t[cut:] for t in expect), "h")


@pytest.mark.parametrize("batch,rows,dim,gates,dtype,gate_dtype", [
    (310, 140, 32, 32, F32, F32), (420, 30, 32, 1, F32, F32), (200, 384, 48, 48, F32, F32), (310, 385, 32, 32, F32, F32),
    (600, 100, 16, 16, F64, F64), (600, 160, 7, 7, F32, F32), (310, 96, 64, 64, BF16, F32), (150, 130, 192, 3, BF16, BF16)])
def test_short_rows_of_many_strips(batch, rows, dim, gates, dtype, gate_dtype):
    """More strips than fit the GPU at once, of few iterations and of one more."""
    run_and_check(make(batch + rows, batch, rows, dim, gates, dtype, gate_dtype, "logit", True), "logit", rows % 2 == 0)


@pytest.mark.parametrize("rows", [200, 3000])  # in one piece and in segments
@pytest.mark.parametrize("dim", [16, 7])
@pytest.mark.parametrize("bad", ["swapped", "outside", "falling", "far", "at the end"])
def test_offsets_that_are_out_of_order_write_nothing_outside(rows, dim, bad):
    """Every output lies between guards, which a row before it or behind it would change."""
    from pysiglib_b200.sequence_inputs import native
    offsets = {"swapped": [0, rows - 50, 50, rows], "outside": [-5, 10, rows + 100], "falling": [rows - 110, 80, 70, 60],
               "far": [2 ** 40, -2 ** 40, 5], "at the end": [rows, rows, rows]}[bad]
    count, guard, kept = len(offsets) - 1, 64 * dim, []

    def guarded(*shape):
        n = int(np.prod(shape))
        kept.append(torch.full((n + 2 * guard,), 7.0, device="cuda"))
        return kept[-1][guard:guard + n].view(shape)
    offsets = torch.tensor(offsets, device="cuda")
    g = torch.Generator().manual_seed(80)
    x, gate, derivs = (torch.rand(rows, dim, generator=g).cuda() for _ in range(3))
    start, tail = (torch.rand(count, dim, generator=g).cuda() for _ in range(2))
    out, state, marks = guarded(rows, dim), guarded(count, dim), guarded(-(-rows // 16), dim)
    dx, dgate, dinitial = guarded(rows, dim), guarded(rows, dim), guarded(count, dim)
    stream, p = torch.cuda.current_stream().cuda_stream, lambda t: t.data_ptr()
    assert native("linear_recurrence")(0, 0, p(x), p(gate), p(start), p(offsets), p(out), p(state), p(marks), 1, rows, dim, dim, count,
                                       0, dim, 0, dim, 0, False, True, -1, stream, 1) == 0
    assert native("linear_recurrence_backprop")(0, 0, p(derivs), p(x), p(gate), p(start), p(offsets), p(tail), p(marks), p(dx), p(dgate),
                                                p(dinitial), 1, rows, dim, dim, count, 0, dim, 0, dim, 0, dim, 0, False, True, -1,
                                                stream, 1) == 0
    for whole in kept:
        assert (whole[:guard] == 7.0).all() and (whole[-guard:] == 7.0).all()
    assert (out != 7.0).all() and (dx != 7.0).all() and (dgate != 7.0).all()  # rows are written whatever the offsets say


def test_a_captured_step_goes_on_with_its_state():
    """Serving: one captured step, replayed for each new row, in inference mode as outside it."""
    x, gate, start, *_ = make(90, 5, 12, 24, 3, BF16, F32, "log", True)
    expect = so.recurrence(x, gate, start, "log", True)
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            X, G, S = cuda(x), cuda(gate), cuda(start)
            row, row_gate = X[:, 0].clone(), G[:, 0].clone()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = psl.linear_recurrence_step(row, row_gate, S, gate_form="log", complement=True)
            for t in range(12):
                row.copy_(X[:, t])
                row_gate.copy_(G[:, t])
                graph.replay()
                so.check(out, (expect["h"][0][:, t], expect["h"][1][:, t]), "row %d" % t)
            so.check(S, expect["state"], "state")


def test_recomputed_and_graphed_layers():
    """The layer under torch's activation checkpointing and as a graphed callable gives the gradients it gives alone."""
    from torch.utils.checkpoint import checkpoint
    x, gate, start, derivs, tail, _ = make(91, 3, 200, 40, 8, F32, F32, "logit", True)

    class Layer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.bias = torch.nn.Parameter(torch.zeros(8, device="cuda"))

        def forward(self, x, gate):
            return torch_api.linear_recurrence(x, gate + self.bias, gate_form="logit", complement=True)

    expect = so.recurrence(x, gate, None, "logit", True, None, derivs)
    layer, X, G = Layer(), cuda(x).requires_grad_(), cuda(gate).requires_grad_()

    def grads(f):
        h = f(X, G)
        so.check(h, expect["h"], "h")
        return torch.autograd.grad(h, (X, G, layer.bias), cuda(derivs))
    # the graphed one first: no eager graph of the same leaves lives beside its capture
    sample = tuple(torch.randn_like(t).requires_grad_() for t in (X, G))
    graphed = torch.cuda.make_graphed_callables(layer, sample)
    for _ in range(2):
        for name, got in zip(("dx", "dgate"), grads(graphed)):
            so.check(got, expect[name], name)
    plain = Layer()
    for f in (plain, lambda x, g: checkpoint(plain, x, g, use_reentrant=False)):
        h = f(X, G)
        dx, dgate, dbias = torch.autograd.grad(h, (X, G, plain.bias), cuda(derivs))
        so.check(dx, expect["dx"], "dx")
        so.check(dgate, expect["dgate"], "dgate")
        assert torch.equal(dbias, dgate.sum((0, 1)))
