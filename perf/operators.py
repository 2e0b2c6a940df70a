"""The sequence operators' cases: gated linear recurrences and rotary positions.

``own`` chooses between the plain form of an operator (elementary torch operations in 32 bits, in 64
for angles and for float64 inputs) and the calls a user makes of pysiglib_b200."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZES = {"float32": 4, "float64": 8, "bfloat16": 2, "float16": 2}


def recurrence(name=None, mode="train", dtype="float32", gate_dtype=None, form="logit", complement=False, batch=1,
               length=1, dim=1, heads=0, sequences=0, initial=False):
    case = {"op": "recurrence", "mode": mode, "dtype": dtype, "gate_dtype": gate_dtype or dtype, "form": form,
            "complement": complement, "batch": batch, "length": length, "dim": dim, "heads": heads or dim,
            "sequences": sequences, "initial": initial}
    return case if name is None else {"name": name, **case}


def rotation(name=None, mode="forward", dtype="bfloat16", batch=1, length=1, heads=1, dim=2, rotary_dim=0,
             interleaved=False, positions="none", rows_first=False):
    case = {"op": "rotary", "mode": mode, "dtype": dtype, "batch": batch, "length": length, "heads": heads, "dim": dim,
            "rotary_dim": rotary_dim or dim, "interleaved": interleaved, "positions": positions,
            "rows_first": rows_first}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # one token for each of 16 streams being served: nothing but latency
        recurrence("step 16x512", "step", "bfloat16", "float32", "log", True, batch=16, dim=512, initial=True),
        # a short path batch of level-4 signatures of 4 channels (340 coefficients), float64
        recurrence("train f64 24x100x340", dtype="float64", form="value", batch=24, length=100, dim=340),
        # windows of a path as a sequence of level-2 signatures of 16 channels (272 coefficients)
        recurrence("train f32 64x512x272", dtype="float32", form="logit", batch=64, length=512, dim=272, initial=True),
        # a layer of ordinary width in training, gates in logits
        recurrence("train bf16 8x4096x2048", dtype="bfloat16", form="logit", complement=True, batch=8, length=4096, dim=2048),
        # one very long path of few channels: the time axis is all there is to split
        recurrence("train f32 1x65536x192", dtype="float32", form="log", batch=1, length=65536, dim=192),
        # packed sequences of different lengths, one gate for 64 channels, log gates kept in float32
        recurrence("train packed 16000x1536", dtype="bfloat16", gate_dtype="float32", form="log", length=16000, dim=1536,
                   heads=24, sequences=23, initial=True),
        # prompts read before serving, packed, with the state kept for the steps that follow
        recurrence("prompt packed 6001x2048", "forward", "float16", "float32", "log", True, length=6001, dim=2048,
                   sequences=7, initial=True),
        # the widest forward pass
        recurrence("forward bf16 8x8192x4096", "forward", "bfloat16", None, "logit", False, batch=8, length=8192, dim=4096),
        # one token for each of 32 streams at its own position
        rotation("rotary step 32x8x128", "forward", "bfloat16", 32, 1, 8, 128, positions="rows"),
        # prompts with heads behind the rows, half of each head kept as it is
        rotation("rotary bf16 4x2048x32x128", "forward", "bfloat16", 4, 2048, 32, 128, 64, positions="rows", rows_first=True),
        # a bank of oscillators at the time stamps of irregularly sampled paths, forward and backward
        rotation("rotary times f32 64x1023x272", "train", "float32", 64, 1023, 1, 272, interleaved=True, positions="times"),
        # a long context
        rotation("rotary bf16 2x32768x16x128", "train", "bfloat16", 2, 32768, 16, 128, rows_first=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.6:
        mode = rng.choice(["train", "train", "forward", "step"])
        dtype = rng.choice(["float32", "float32", "bfloat16", "float16", "float64"])
        gate_dtype = "float32" if dtype in ("bfloat16", "float16") and rng.random() < 0.5 else dtype
        group = rng.choice([1, 1, 1, 16, 64, 128])
        heads = max(1, _spread(rng, 5, 4096) // group)
        dim = heads * group
        shared = heads if group > 1 else 0
        form, complement, initial = rng.choice(["value", "log", "logit"]), rng.random() < 0.4, rng.random() < 0.5
        if mode == "step":
            return recurrence(None, mode, dtype, gate_dtype, form, complement, _spread(rng, 1, 512), 1, dim, shared, 0, True)
        length = _spread(rng, 1, 65536)
        batch = _spread(rng, 1, max(1, min(256, (1 << 25) // (dim * length))))
        sequences = rng.choice([0, 0, _spread(rng, 1, 64)])
        if sequences:
            length, batch = length * batch, 1
        return _within(recurrence(None, mode, dtype, gate_dtype, form, complement, batch, length, dim, shared,
                                  sequences, initial))
    dim = rng.choice([16, 32, 64, 64, 80, 96, 128, 128, 256, 2 * _spread(rng, 2, 300)])
    part = rng.choice([dim, dim, 2 * max(1, dim // 4), 2 * rng.randint(1, dim // 2)])
    length, heads = _spread(rng, 1, 65536), rng.choice([1, 2, 4, 8, 12, 16, 32])
    batch = _spread(rng, 1, max(1, min(256, (1 << 26) // (dim * length * heads))))
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32", "float64"])
    return _within(rotation(None, rng.choice(["forward", "train"]), dtype, batch, length, heads, dim, part,
                            rng.random() < 0.4, rng.choice(["none", "rows", "times"]), rng.random() < 0.5))


def _within(case):
    """The case, shortened until it moves no more than the listed ones."""
    while work(case)["bytes"] > 1.0e9:
        case["length"] = max(1, case["length"] // 2)
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "rotary":
        shape = ((case["batch"], case["length"], case["heads"], case["dim"]) if case["rows_first"] else
                 (case["batch"], case["heads"], case["length"], case["dim"]))
        state = {"case": case, "x": normal(*shape).to(dtype), "positions": None}
        if case["rows_first"]:
            state["x"] = state["x"].transpose(1, 2)
        half = case["rotary_dim"] // 2
        state["frequencies"] = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        if case["positions"] == "rows":  # each stream at its own place in a context of up to 131072 tokens
            start = torch.randint(0, 131072 - case["length"], (case["batch"], 1), generator=g, device="cuda")
            state["positions"] = (start + torch.arange(case["length"], device="cuda")).unsqueeze(1)
        elif case["positions"] == "times":
            gaps = torch.rand(case["batch"], 1, case["length"], generator=g, device="cuda", dtype=torch.float64)
            state["positions"] = torch.cumsum(2.0 * gaps, -1)
        if case["mode"] == "train":
            state["derivs"] = normal(*shape).to(dtype)
            if case["rows_first"]:
                state["derivs"] = state["derivs"].transpose(1, 2)
        return state

    lead = () if case["sequences"] else (case["batch"],)
    rows = () if case["mode"] == "step" else (case["length"],)
    wide = torch.float64 if dtype is torch.float64 else torch.float32
    state = {"case": case, "x": normal(*lead, *rows, case["dim"]).to(dtype), "initial": None, "offsets": None}
    # gates between about 0.5 and 0.998: memories of a few tokens to some hundreds
    logits = 3.0 + 1.5 * normal(*lead, *rows, case["heads"]).clamp(-2, 2)
    gate = {"value": torch.sigmoid, "log": torch.nn.functional.logsigmoid, "logit": lambda v: v}[case["form"]](logits)
    state["gate"] = gate.to(DTYPES[case["gate_dtype"]])
    if case["sequences"]:
        cuts = torch.randint(0, case["length"] + 1, (case["sequences"] - 1,), generator=g, device="cuda").sort().values
        ends = torch.tensor([0, case["length"]], device="cuda")
        state["offsets"] = torch.cat([ends[:1], cuts, ends[1:]])
    if case["initial"]:
        count = (case["sequences"],) if case["sequences"] else (case["batch"],)
        state["initial"] = normal(*count, case["dim"]).to(wide)
    if case["mode"] == "train":
        state["derivs"] = normal(*lead, *rows, case["dim"]).to(dtype)
    return state


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        return run_rotary(state)
    return run_step(state) if case["mode"] == "step" else run_recurrence(state)


def run_step(state):
    case = state["case"]
    if own:
        import pysiglib_b200 as psl
        out = psl.linear_recurrence_step(state["x"], state["gate"], state["initial"], gate_form=case["form"],
                                         complement=case["complement"])
        return {"out": out, "state": state["initial"]}
    a, rest = plain_gate(state["gate"], case, state["initial"].dtype)
    x = state["x"].to(state["initial"].dtype)
    state["initial"].copy_(a * state["initial"] + (rest * x if case["complement"] else x))
    return {"out": state["initial"].to(state["x"].dtype), "state": state["initial"]}


def run_recurrence(state):
    case = state["case"]
    if own:
        import pysiglib_b200 as psl
        how = {"gate_form": case["form"], "complement": case["complement"], "offsets": state["offsets"]}
        if case["mode"] == "forward":
            h, last = psl.linear_recurrence(state["x"], state["gate"], state["initial"], return_state=True, **how)
            return {"h": h, "state": last}
        h, last, marks = psl.linear_recurrence(state["x"], state["gate"], state["initial"], return_state=True,
                                               return_checkpoints=True, **how)
        result = {"h": h, "state": last}
        result["dx"], result["dgate"], result["dinitial"] = psl.linear_recurrence_backprop(
            state["derivs"], state["x"], state["gate"], state["initial"], checkpoints=marks, **how)
        return result
    dtype = state["x"].dtype
    wide = torch.float64 if dtype is torch.float64 else torch.float32
    a, rest = plain_gate(state["gate"], case, wide)
    x = state["x"].to(wide)
    b = rest * x if case["complement"] else x
    axis = x.dim() - 2
    starts, of_row, first, last, empty = plain_sequences(state)
    held = b.new_zeros((case["sequences"] or case["batch"], case["dim"])) if state["initial"] is None else state["initial"]
    entering = of_row(held)
    # the state that enters a sequence becomes part of its first row, whose gate then lets nothing else in
    b = torch.where(starts, b + a * entering, b)
    cut = torch.where(starts, 0.0, a)
    h = plain_scan(cut, b, axis)
    result = {"h": h.to(dtype), "state": torch.where(empty, held, last(h))}
    if case["mode"] == "train":
        edge = torch.zeros_like(h.narrow(axis, 0, 1))
        before = torch.where(starts, entering, torch.cat([edge, h.narrow(axis, 0, h.shape[axis] - 1)], axis))
        # g_t = dh_t + a_{t+1} g_{t+1}: the same scan from the other end, with the gates one row further
        after = torch.cat([cut.narrow(axis, 1, h.shape[axis] - 1), edge], axis)
        g = plain_scan(after.flip(axis), state["derivs"].to(wide).flip(axis), axis).flip(axis)
        da = g * (before - x) if case["complement"] else g * before
        slope = {"value": None, "log": a, "logit": a * rest}[case["form"]]
        dgate = da if slope is None else da * slope
        if case["heads"] != case["dim"]:
            dgate = dgate.unflatten(-1, (case["heads"], -1)).sum(-1)
        result["dx"] = (rest * g if case["complement"] else g).to(dtype)
        result["dgate"] = dgate.to(state["gate"].dtype)
        result["dinitial"] = None if state["initial"] is None else torch.where(empty, 0.0, first(a * g))
    return result


def plain_gate(gate, case, wide):
    """a and 1 - a, each without cancellation, on all channels."""
    v = gate.to(wide)
    a, rest = {"value": lambda: (v, 1 - v), "log": lambda: (torch.exp(v), -torch.expm1(v)),
               "logit": lambda: (1 / (1 + torch.exp(-v)), 1 / (1 + torch.exp(v)))}[case["form"]]()
    if case["heads"] != case["dim"]:
        a, rest = (t.repeat_interleave(case["dim"] // case["heads"], -1) for t in (a, rest))
    return a, rest


def plain_sequences(state):
    """Which rows start a sequence, the sequences' values on their rows, the rows' values at the
    sequences' first and last rows, and which sequences are empty."""
    offsets, x = state["offsets"], state["x"]
    if offsets is None:
        rows = torch.arange(x.shape[1], device="cuda").unsqueeze(-1)
        return rows == 0, lambda held: held.unsqueeze(1), lambda t: t[:, 0], lambda t: t[:, -1], (rows[:1] < 0)[0]
    rows = torch.arange(x.shape[0], device="cuda")
    owner = torch.searchsorted(offsets, rows, right=True) - 1
    begin, end = offsets[:-1].clamp(max=x.shape[0] - 1), (offsets[1:] - 1).clamp(min=0)
    return ((offsets[owner] == rows).unsqueeze(-1), lambda held: held[owner], lambda t: t[begin], lambda t: t[end],
            (offsets[1:] == offsets[:-1]).unsqueeze(-1))


def plain_scan(a, b, axis):
    """h_t = a_t h_{t-1} + b_t by doubling: after the pass with step s every row holds its last 2 s rows."""
    step, n = 1, a.shape[axis]
    while step < n:
        tail_a, tail_b = a.narrow(axis, step, n - step), b.narrow(axis, step, n - step)
        b = torch.cat([b.narrow(axis, 0, step), tail_b + tail_a * b.narrow(axis, 0, n - step)], axis)
        a = torch.cat([a.narrow(axis, 0, step), tail_a * a.narrow(axis, 0, n - step)], axis)
        step *= 2
    return b


def run_rotary(state):
    case, x = state["case"], state["x"]
    if own:
        import pysiglib_b200 as psl
        how = {"interleaved": case["interleaved"]}
        result = {"y": psl.rotary(x, state["frequencies"], state["positions"], **how)}
        if case["mode"] == "train":
            result["dx"] = psl.rotary_backprop(state["derivs"], state["frequencies"], state["positions"], **how)
        return result
    wide = torch.float64 if x.dtype is torch.float64 else torch.float32
    positions = state["positions"]
    if positions is None:
        positions = torch.arange(case["length"], device="cuda")
    angles = positions.to(torch.float64).unsqueeze(-1) * state["frequencies"]
    cos, sin = torch.cos(angles).to(wide), torch.sin(angles).to(wide)
    result = {"y": plain_rotation(x, cos, sin, case, wide)}
    if case["mode"] == "train":
        result["dx"] = plain_rotation(state["derivs"], cos, -sin, case, wide)
    return result


def plain_rotation(x, cos, sin, case, wide):
    part = case["rotary_dim"]
    v = x[..., :part].to(wide)
    p, q = (v[..., 0::2], v[..., 1::2]) if case["interleaved"] else (v[..., :part // 2], v[..., part // 2:])
    y = (p * cos - q * sin, p * sin + q * cos)
    y = torch.stack(y, -1).flatten(-2) if case["interleaved"] else torch.cat(y, -1)
    return torch.cat([y.to(x.dtype), x[..., part:]], -1)


def work(case):
    size, gate_size = SIZES[case["dtype"]], SIZES[case.get("gate_dtype", case["dtype"])]
    train = case["mode"] == "train"
    if case["op"] == "rotary":
        n = case["batch"] * case["heads"] * case["length"] * case["dim"]
        return {"bytes": (4 if train else 2) * n * size, "flops": (6 if train else 3) * n}
    rows = case["batch"] * case["length"]
    n, gates = rows * case["dim"], rows * case["heads"]
    held = (case["sequences"] or case["batch"]) * case["dim"] * max(size, 4)
    count = 2 * n * size + gates * gate_size + held * (2 if case["initial"] else 1)
    if train:  # derivatives, inputs and gates in, two gradients out (and those of the initial states)
        count += 3 * n * size + 2 * gates * gate_size + (2 * held if case["initial"] else 0)
    return {"bytes": count, "flops": (7 if train else 2) * n}


def exact(case, seed):
    """The definitions row by row in 64 bits."""
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return exact_rotary(case, state)
    x, v = state["x"].double(), state["gate"].double().repeat_interleave(case["dim"] // case["heads"], -1)
    a = {"value": lambda: v, "log": lambda: torch.exp(v), "logit": lambda: torch.sigmoid(v)}[case["form"]]()
    rest = {"value": lambda: 1 - v, "log": lambda: -torch.expm1(v), "logit": lambda: torch.sigmoid(-v)}[case["form"]]()
    b = rest * x if case["complement"] else x
    if case["mode"] == "step":
        h = a * state["initial"].double() + b
        return {"out": h, "state": h}
    if case["sequences"]:
        spans = state["offsets"].tolist()
        spans = list(zip(spans[:-1], spans[1:]))
        a, rest, b, x = (t.unsqueeze(1) for t in (a, rest, b, x))
    else:
        spans = [(0, case["length"])]
        a, rest, b, x = (t.transpose(0, 1).contiguous() for t in (a, rest, b, x))
    derivs = None
    if case["mode"] == "train":
        d = state["derivs"].double()
        derivs = d.unsqueeze(1) if case["sequences"] else d.transpose(0, 1).contiguous()
    h, before, finals = torch.empty_like(b), torch.empty_like(b), []
    g, entered = torch.empty_like(b), []
    for k, (start, end) in enumerate(spans):
        now = torch.zeros_like(b[:1].sum(0))
        if case["initial"]:
            now = state["initial"][k:k + 1].double() if case["sequences"] else state["initial"].double()
        for t in range(start, end):
            before[t].copy_(now)
            now = torch.addcmul(b[t], a[t], now, out=h[t])
        finals.append(now.clone())
        if derivs is not None:
            back = torch.zeros_like(now)
            for t in range(end - 1, start - 1, -1):
                torch.add(derivs[t], back, out=g[t])
                back = a[t] * g[t]
            entered.append(back)

    def shaped(t):
        return t.squeeze(1) if case["sequences"] else t.transpose(0, 1)

    def joined(ts):
        return torch.cat(ts) if case["sequences"] else ts[0]

    result = {"h": shaped(h), "state": joined(finals)}
    if derivs is not None:
        da = g * before - (g * x if case["complement"] else 0)
        da = da * {"value": lambda: 1.0, "log": lambda: a, "logit": lambda: a * rest}[case["form"]]()
        if case["heads"] != case["dim"]:
            da = da.reshape(*da.shape[:-1], case["heads"], -1).sum(-1)
        result["dx"] = shaped(rest * g if case["complement"] else g)
        result["dgate"] = shaped(da)
        result["dinitial"] = joined(entered) if case["initial"] else None
    return result


def exact_rotary(case, state):
    half = case["rotary_dim"] // 2
    positions = torch.arange(case["length"], device="cuda") if state["positions"] is None else state["positions"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       positions.double()[..., None] * state["frequencies"])

    def turned(x, by):
        y = x.double().clone()
        if case["interleaved"]:
            real, imag = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        else:
            real, imag = slice(0, half), slice(half, 2 * half)
        z = torch.complex(y[..., real], y[..., imag]) * by
        y[..., real], y[..., imag] = z.real, z.imag
        return y

    result = {"y": turned(state["x"], turn)}
    if case["mode"] == "train":
        result["dx"] = turned(state["derivs"], turn.conj())
    return result
