"""The short causal convolution and the selective scan of state-space layers against statements in 64 bits.

Tolerances count roundings: half a step relative to the value is 2^-24 in float32 and 2^-8 in bfloat16.  CUDA documents its
exponential as off by at most 1 step of float32 for ``expf`` and 2^-22.5 (relative) for the approximate exponential of base two; the
bounds below allow 2^-21 for an exponential and 2^-21 for a silu or softplus made from one (a sum, a logarithm or quotient more).
"""
from types import SimpleNamespace

import pytest
import torch

from oxidize_b200 import ops

HALF = 2.0 ** -24  # of float32, relative
EXP = 2.0 ** -21  # of an exponential, silu or softplus, relative
BF16 = 2.0 ** -8
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def step(lens, device, fresh=None, no_slot=(), slots=None, seed=0):
    """A step that feeds ``lens`` rows; sequences in ``fresh`` start at position 0."""
    gen = torch.Generator().manual_seed(seed)
    B = len(lens)
    before = [0 if (i % 2 == 0 if fresh is None else i in fresh) else int(torch.randint(1, 40, (1,), generator=gen)) for i in range(B)]
    at = torch.randperm(B + 2, generator=gen)[:B].tolist() if slots is None else list(slots)
    for i in no_slot:
        at[i] = -1
    start = [0]
    for n in lens:
        start.append(start[-1] + n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    return SimpleNamespace(query_start=i32(start), seq_lens=i32([b + n for b, n in zip(before, lens)]), state_slots=i32(at),
                           max_query_len=max(lens + [1]), host_lens=[(n, b + n) for b, n in zip(before, lens)])


def rows(gen, T, C, dtype, device, wide=0, off=0, scale=1.0):
    """[T, C] columns of a matrix ``wide`` columns wider, from column ``off``."""
    m = (torch.randn(T, C + wide, generator=gen) * scale).to(dtype).to(device)
    return m[:, off : off + C]


def out_bound(y, err, dtype):
    return err if dtype == torch.float32 else err + BF16 * (y.abs() + err)


# --------------------------------------------------------------------------------------------------------- convolution
def conv64(x, w, bias, meta, window, act):
    """(y, bound of float32's roundings, window, rows that belong to a sequence with a slot) in 64 bits."""
    T, C = x.shape
    K = w.shape[1]
    x, w, win = x.double(), w.double(), window.double().clone()
    y, size = torch.zeros(T, C, dtype=torch.float64, device=x.device), torch.zeros(T, C, dtype=torch.float64, device=x.device)
    qs, lens, slots = meta.query_start.tolist(), meta.seq_lens.tolist(), meta.state_slots.tolist()
    for b, s in enumerate(slots):
        n = qs[b + 1] - qs[b]
        if s < 0:
            continue
        pos0 = lens[b] - n
        value = lambda p: x[qs[b] + p - pos0] if p >= pos0 else (window[s, p % K].double() if p >= 0 else torch.zeros_like(x[0]))  # noqa: E731
        for j in range(n):
            t = qs[b] + j
            terms = torch.stack([w[:, i] * value(pos0 + j - (K - 1) + i) for i in range(K)])
            y[t] = terms.sum(0) + (0 if bias is None else bias.double())
            size[t] = terms.abs().sum(0) + (0 if bias is None else bias.double().abs())
        for j in range(max(0, n - K), n):
            win[s, (pos0 + j) % K] = x[qs[b] + j]
    err = (K + 1) * HALF * size  # of K products that are added up, and the bias
    if act == "silu":
        err = 1.1 * err  # the steepest slope of silu
        y = y * torch.sigmoid(y)
        err = err + EXP * y.abs()
    return y, err, win


CONVS = [
    # lens, channels, taps, type, out, act, bias, wide, off
    ([1], 64, 4, "bf16", "f32", "silu", True, 0, 0),
    ([1, 1, 1, 1, 1], 130, 4, "bf16", "f32", "silu", True, 130, 0),
    ([1] * 40, 72, 3, "f32", "bf16", "none", True, 72, 72),
    ([5, 0, 1, 17, 2, 3], 33, 4, "bf16", "bf16", "silu", True, 7, 1),
    ([0, 0, 3], 8, 4, "f32", "f32", "silu", False, 0, 0),
    ([65, 64, 63], 256, 4, "bf16", "f32", "silu", True, 256, 0),
    ([130], 1, 2, "f32", "f32", "silu", True, 0, 0),
    ([300, 1, 9], 520, 8, "bf16", "f32", "none", False, 8, 8),
    ([37, 40], 12, 1, "bf16", "f32", "silu", True, 0, 0),
    ([20, 31], 19, 5, "f32", "f32", "silu", True, 4, 3),
    ([2, 2, 2, 2, 3, 1, 1], 1000, 4, "bf16", "f32", "silu", True, 1000, 0),
]
TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", CONVS, ids=[str(i) for i in range(len(CONVS))])
def test_convolution(case, device):
    lens, C, K, kind, out, act, with_bias, wide, off = case
    gen = torch.Generator().manual_seed(3)
    meta = step(lens, device)
    x = rows(gen, sum(lens), C, TYPE[kind], device, wide, off)
    w, bias = torch.randn(C, K, generator=gen).to(device), torch.randn(C, generator=gen).to(device) if with_bias else None
    window = torch.randn(len(lens) + 2, K, C, generator=gen).to(device)
    want, err, after = conv64(x, w, bias, meta, window, act)
    y = ops.causal_conv(x, w, bias, meta, window, act=act, act_dtype=TYPE[out])
    assert y.dtype == TYPE[out]
    assert ((y.double() - want).abs() <= out_bound(want, err, TYPE[out])).all()
    assert torch.equal(window.double(), after)


@pytest.mark.parametrize("device", DEVICES)
def test_convolution_leaves_other_rows_and_slots_alone(device):
    """Rows behind the last sequence stay as they were, those of a sequence without a slot become zeros, other slots stay."""
    gen = torch.Generator().manual_seed(5)
    lens, C, K = [3, 4, 1], 40, 4
    meta = step(lens, device, no_slot=(1,), slots=(4, 0, 2))
    x = rows(gen, 12, C, torch.bfloat16, device)  # four rows more than the sequences have
    w, window = torch.randn(C, K, generator=gen).to(device), torch.randn(6, K, C, generator=gen).to(device)
    before, wide = window.clone(), torch.full((12, 2 * C), 7.0, device=device)
    out = wide[:, 3 : 3 + C]
    want, err, after = conv64(x[:8], w, None, meta, window, "silu")
    assert ops.causal_conv(x, w, None, meta, window, out=out) is out
    assert ((out[:8].double() - want).abs() <= err).all() and (out[3:7] == 0).all()
    assert (wide[8:] == 7).all() and (wide[:, :3] == 7).all() and (wide[:, 3 + C :] == 7).all()
    assert torch.equal(window.double(), after) and torch.equal(window[[0, 1, 3, 5]], before[[0, 1, 3, 5]])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cuts", [[20], [1] * 20, [7, 13], [3, 1, 1, 9, 6], [19, 1]])
def test_convolution_of_portions_is_the_whole(cuts, device):
    """The same bits whatever portions a sequence comes in, next to another sequence."""
    gen = torch.Generator().manual_seed(6)
    C, K = 72, 4
    x, w = rows(gen, 20, C, torch.bfloat16, device), torch.randn(C, K, generator=gen).to(device)
    bias = torch.randn(C, generator=gen).to(device)

    def feed(parts):
        window, at, got = torch.full((2, K, C), 9.0, device=device), 0, []
        for n in parts:
            meta = step([2, n], device, slots=(0, 1))
            meta.seq_lens[1] = at + n
            y = ops.causal_conv(torch.cat([x[:2], x[at : at + n]]), w, bias, meta, window)
            got.append(y[2:])
            at += n
        return torch.cat(got), window[1]

    y, window = feed(cuts)
    whole, end = feed([20])
    assert torch.equal(window, end)
    # (the CPU takes vector and scalar forms of silu in turn, each within EXP of the same sum's)
    assert torch.equal(y, whole) if device == "cuda" else ((y - whole).abs() <= 2 * EXP * whole.abs()).all()


@pytest.mark.parametrize("device", DEVICES)
def test_convolution_keeps_what_is_not_finite_to_its_channel(device):
    gen = torch.Generator().manual_seed(7)
    lens, C, K = [6, 9, 1], 24, 4
    meta = step(lens, device, fresh=(0, 1))
    x = rows(gen, 16, C, torch.float32, device)
    w, window = torch.randn(C, K, generator=gen).to(device), torch.randn(5, K, C, generator=gen).to(device)
    window[meta.state_slots[:2].long()] = float("nan")  # of sequences that start: not read
    clean = ops.causal_conv(x, w, None, meta, window.clone(), act="none")
    x[8, 5], x[2, 1] = float("inf"), float("nan")
    y = ops.causal_conv(x, w, None, meta, window, act="none")
    touched = torch.zeros(16, C, dtype=torch.bool, device=device)
    touched[8:12, 5] = touched[2:6, 1] = True
    assert torch.isfinite(clean).all() and torch.equal(y[~touched], clean[~touched]) and not torch.isfinite(y[touched]).any()


# ---------------------------------------------------------------------------------------------------------------- scan
def scan64(u, dt, a, b, c, d, z, dt_bias, meta, state):
    """(y, bound of float32's roundings, state, its bound) in 64 bits."""
    T, C = u.shape
    u, dt, a, b, c = (v.double() for v in (u, dt, a, b, c))
    raw = dt if dt_bias is None else dt + dt_bias.double()
    s = torch.logaddexp(raw, torch.zeros_like(raw))
    # the sum's rounding (slope of softplus at most 1; relative to what is left of it: e^x where x is very negative) and its own
    s_err = s * (HALF * (dt.abs() + raw.abs()) + EXP)
    y, err = torch.zeros(T, C, dtype=torch.float64, device=u.device), torch.zeros(T, C, dtype=torch.float64, device=u.device)
    after, after_err = state.double().clone(), torch.zeros_like(state, dtype=torch.float64)
    qs, lens, slots = meta.query_start.tolist(), meta.seq_lens.tolist(), meta.state_slots.tolist()
    for i, slot in enumerate(slots):
        t0, t1 = qs[i], qs[i + 1]
        if slot < 0 or t0 == t1:
            continue
        h = torch.zeros(a.shape, dtype=torch.float64, device=u.device) if lens[i] == t1 - t0 else state[slot].double()
        e = torch.zeros_like(h)
        for t in range(t0, t1):
            x = s[t][:, None] * a
            keep, add = torch.exp(x), (s[t] * u[t])[:, None] * b[t]
            # of the exponent (a and the product are rounded when its base becomes two: three roundings) and the exponential
            keep_err = keep * (s_err[t][:, None] * a.abs() + 3 * HALF * x.abs() + EXP)
            add_err = (s_err[t] * u[t].abs())[:, None] * b[t].abs() + 2 * HALF * add.abs()
            e = (keep + keep_err) * e + h.abs() * keep_err + add_err
            h = keep * h + add
            e = e + HALF * h.abs() + HALF * e
            y[t] = (h * c[t]).sum(1) + (0 if d is None else d.double() * u[t])
            size = (h * c[t]).abs().sum(1) + (0 if d is None else (d.double() * u[t]).abs())
            err[t] = (e * c[t].abs()).sum(1) + (a.shape[1] + 1) * HALF * size
        after[slot], after_err[slot] = h, e
    if z is not None:
        gate = z.double() * torch.sigmoid(z.double())
        y, err = y * gate, (err + (EXP + HALF) * y.abs()) * gate.abs()
    return y, err * (1 + 1e-6) + 1e-37, after, after_err * (1 + 1e-6) + 1e-37


SCANS = [
    # lens, channels, states, types of u, dt, (b, c), out; gate, d, dt_bias, wide
    ([1], 64, 16, "f32", "f32", "f32", "bf16", True, True, True, 0),
    ([1] * 33, 130, 16, "f32", "f32", "f32", "bf16", True, True, True, 8),
    ([1, 1, 1], 5, 1, "bf16", "f32", "bf16", "f32", False, False, False, 0),
    ([5, 0, 1, 17, 2], 33, 16, "bf16", "bf16", "bf16", "bf16", True, True, True, 5),
    ([70, 64, 31], 96, 16, "f32", "f32", "f32", "f32", True, True, True, 96),
    ([40], 1, 8, "f32", "f32", "f32", "f32", True, True, False, 0),
    ([33, 2], 20, 5, "f32", "bf16", "f32", "f32", False, True, True, 3),
    ([19, 40], 17, 17, "bf16", "f32", "f32", "bf16", True, False, True, 0),
    ([21], 40, 64, "f32", "f32", "f32", "f32", True, True, True, 0),
    ([1, 18], 24, 128, "f32", "f32", "bf16", "f32", True, True, True, 4),
    ([100], 300, 16, "f32", "f32", "f32", "bf16", True, True, True, 300),
    ([0, 16, 32], 64, 2, "f32", "f32", "f32", "f32", False, True, True, 0),
]


def scan_inputs(gen, T, C, N, tu, tdt, tbc, tout, gate, with_d, with_bias, wide, device):
    par = rows(gen, T, 2 * N, TYPE[tbc], device, 3, 1)
    return dict(u=rows(gen, T, C, TYPE[tu], device, wide), dt=rows(gen, T, C, TYPE[tdt], device, wide, wide),
                a=(-torch.rand(C, N, generator=gen) * 16).to(device), b=par[:, :N], c=par[:, N:],
                d=torch.randn(C, generator=gen).to(device) if with_d else None,
                z=rows(gen, T, C, TYPE[tout], device, C, C) if gate else None,
                dt_bias=(torch.randn(C, generator=gen) - 3).to(device) if with_bias else None)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", SCANS, ids=[str(i) for i in range(len(SCANS))])
def test_scan(case, device):
    lens, C, N, tu, tdt, tbc, tout, gate, with_d, with_bias, wide = case
    gen = torch.Generator().manual_seed(11)
    meta = step(lens, device)
    v = scan_inputs(gen, sum(lens), C, N, tu, tdt, tbc, tout, gate, with_d, with_bias, wide, device)
    state = torch.randn(len(lens) + 2, C, N, generator=gen).to(device)
    want, err, after, after_err = scan64(**v, meta=meta, state=state)
    y = ops.selective_scan(**v, meta=meta, state=state, act_dtype=TYPE[tout])
    assert y.dtype == TYPE[tout]
    assert ((y.double() - want).abs() <= out_bound(want, err, TYPE[tout])).all()
    assert ((state.double() - after).abs() <= after_err).all()


@pytest.mark.parametrize("device", DEVICES)
def test_scan_leaves_other_rows_and_slots_alone(device):
    gen = torch.Generator().manual_seed(12)
    lens, C, N = [3, 4, 1], 40, 16
    meta = step(lens, device, no_slot=(1,), slots=(4, 0, 2))
    v = scan_inputs(gen, 12, C, N, "f32", "f32", "f32", "bf16", True, True, True, 0, device)
    # one layer's slots among several layers'
    state = torch.randn(6, 3, C, N, generator=gen).to(device)
    before, wide = state.clone(), torch.full((12, 2 * C), 7.0, dtype=torch.bfloat16, device=device)
    out = wide[:, 5 : 5 + C]
    want, err, after, after_err = scan64(**v, meta=meta, state=state[:, 1])
    assert ops.selective_scan(**v, meta=meta, state=state[:, 1], act_dtype=torch.bfloat16, out=out) is out
    assert ((out[:8].double() - want[:8]).abs() <= out_bound(want, err, torch.bfloat16)[:8]).all() and (out[3:7] == 0).all()
    assert (wide[8:] == 7).all() and (wide[:, :5] == 7).all() and (wide[:, 5 + C :] == 7).all()
    assert ((state[:, 1].double() - after).abs() <= after_err).all()
    assert torch.equal(state[:, [0, 2]], before[:, [0, 2]]) and torch.equal(state[[0, 1, 3, 5]], before[[0, 1, 3, 5]])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("C,N", [(72, 16), (2600, 16), (9, 40)])
@pytest.mark.parametrize("cuts", [[1] * 40, [7, 33], [16, 16, 8], [39, 1]])
def test_scan_of_portions_is_the_whole(cuts, C, N, device):
    """The same bits whatever portions a sequence comes in, and whatever runs beside it."""
    gen = torch.Generator().manual_seed(13)
    v = scan_inputs(gen, 40, C, N, "f32", "f32", "f32", "f32", True, True, True, 0, device)

    def feed(parts, beside):
        state, at, got = torch.full((3, C, N), 9.0, device=device), 0, []
        for n in parts:
            meta = step([beside, n], device, slots=(0, 2))
            meta.seq_lens[1] = at + n
            take = torch.cat([torch.arange(beside), torch.arange(at, at + n)]).to(device)
            part = {k: x[take] if k in ("u", "dt", "b", "c", "z") else x for k, x in v.items()}
            got.append(ops.selective_scan(**part, meta=meta, state=state)[beside:])
            at += n
        return torch.cat(got), state[2]

    y, state = feed(cuts, 2)
    whole, end = feed([40], 0)
    if device == "cuda":
        assert torch.equal(y, whole) and torch.equal(state, end)
    else:  # (the CPU takes vector and scalar forms of its functions in turn: both within the bound)
        meta = step([40], device, slots=(2,), fresh=(0,))
        want, err, after, after_err = scan64(**v, meta=meta, state=torch.zeros(3, C, N))
        for got, kept in ((y, state), (whole, end)):
            assert ((got.double() - want).abs() <= err).all() and ((kept.double() - after[2]).abs() <= after_err[2]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_scan_with_steps_far_from_one(device):
    """Steps so large that softplus is the identity and nothing is kept, or so small that nothing happens; a state of zeros."""
    gen = torch.Generator().manual_seed(14)
    meta = step([30], device, fresh=())
    v = scan_inputs(gen, 30, 24, 16, "f32", "f32", "f32", "f32", True, True, False, 0, device)
    v["dt"][:, :8] = 60.0
    v["dt"][:, 8:16] = -120.0
    state = torch.randn(3, 24, 16, generator=gen).to(device)
    want, err, after, after_err = scan64(**v, meta=meta, state=state)
    y = ops.selective_scan(**v, meta=meta, state=state)
    assert ((y.double() - want).abs() <= err).all() and ((state.double() - after).abs() <= after_err).all()


@pytest.mark.parametrize("device", DEVICES)
def test_scan_keeps_what_is_not_finite_to_its_channel(device):
    gen = torch.Generator().manual_seed(15)
    lens, C, N = [6, 9, 1], 24, 16
    meta = step(lens, device, fresh=(0, 1))
    v = scan_inputs(gen, 16, C, N, "f32", "f32", "f32", "f32", True, True, True, 0, device)
    state = torch.randn(5, C, N, generator=gen).to(device)
    state[meta.state_slots[:2].long()] = float("nan")  # of sequences that start: not read
    clean = ops.selective_scan(**v, meta=meta, state=state.clone())
    v["u"][8, 5] = float("nan")
    y = ops.selective_scan(**v, meta=meta, state=state)
    touched = torch.zeros(16, C, dtype=torch.bool, device=device)
    touched[8:15, 5] = True
    assert torch.isfinite(clean).all() and torch.equal(y[~touched], clean[~touched]) and torch.isnan(y[touched]).all()
    assert torch.isfinite(state[meta.state_slots[[0, 2]].long()]).all()


# ------------------------------------------------------------------------------------------------------------ refusals
def _scan_call(device, **change):
    gen = torch.Generator().manual_seed(1)
    v = dict(scan_inputs(gen, 4, 8, 16, "f32", "f32", "f32", "f32", True, True, True, 0, device), meta=step([4], device),
             state=torch.zeros(3, 8, 16, device=device))
    v.update({k: f(v) for k, f in change.items()})
    return ops.selective_scan(**v)


def _conv_call(device, **change):
    gen = torch.Generator().manual_seed(1)
    v = dict(x=rows(gen, 4, 8, torch.float32, device), w=torch.zeros(8, 4, device=device), bias=torch.zeros(8, device=device),
             meta=step([4], device), window=torch.zeros(3, 4, 8, device=device))
    v.update({k: f(v) for k, f in change.items()})
    return ops.causal_conv(**v)


def _without_slots(v):
    v["meta"].state_slots = None
    return v["meta"]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("call,change", [
    (_scan_call, dict(dt=lambda v: v["dt"][:, :7])), (_scan_call, dict(dt=lambda v: v["dt"][:3])),
    (_scan_call, dict(b=lambda v: v["b"][:, :15])), (_scan_call, dict(c=lambda v: v["c"][:3])),
    (_scan_call, dict(a=lambda v: v["a"][:7])), (_scan_call, dict(z=lambda v: v["z"][:, :4])),
    (_scan_call, dict(d=lambda v: v["d"][:4])), (_scan_call, dict(dt_bias=lambda v: v["dt_bias"][:, None])),
    (_scan_call, dict(state=lambda v: v["state"][:, :, :8])), (_scan_call, dict(state=lambda v: v["state"].double())),
    (_scan_call, dict(state=lambda v: v["state"][0])), (_scan_call, dict(meta=_without_slots)),
    (_conv_call, dict(w=lambda v: v["w"][:7])), (_conv_call, dict(w=lambda v: v["w"][:, :3])),
    (_conv_call, dict(bias=lambda v: v["bias"][:7])), (_conv_call, dict(window=lambda v: v["window"][:, :3])),
    (_conv_call, dict(window=lambda v: v["window"].bfloat16())), (_conv_call, dict(act=lambda v: "gelu")),
    (_conv_call, dict(meta=_without_slots))])
def test_what_does_not_fit_is_refused(call, change, device):
    call(device)
    with pytest.raises(ValueError):
        call(device, **change)


@pytest.mark.gpu
@pytest.mark.parametrize("call,change", [
    (_scan_call, dict(u=lambda v: v["u"].half())), (_scan_call, dict(b=lambda v: v["b"].double())),
    (_scan_call, dict(a=lambda v: v["a"].bfloat16())), (_scan_call, dict(act_dtype=lambda v: torch.float16)),
    (_scan_call, dict(state=lambda v: torch.zeros(3, 16, 8, device="cuda").transpose(1, 2))),
    (_scan_call, dict(out=lambda v: torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda"))),
    (_scan_call, dict(out=lambda v: torch.zeros(3, 8, device="cuda"))),
    (_scan_call, dict(a=lambda v: torch.zeros(8, 129, device="cuda"), b=lambda v: torch.zeros(4, 129, device="cuda"),
                      c=lambda v: torch.zeros(4, 129, device="cuda"), state=lambda v: torch.zeros(3, 8, 129, device="cuda"))),
    (_conv_call, dict(x=lambda v: v["x"].half())), (_conv_call, dict(w=lambda v: v["w"].double())),
    (_conv_call, dict(window=lambda v: torch.zeros(3, 8, 4, device="cuda").transpose(1, 2))),
    (_conv_call, dict(out=lambda v: torch.zeros(8, 4, device="cuda").t()))])
def test_what_the_kernels_do_not_read_is_refused(call, change):
    with pytest.raises(ValueError):
        call("cuda", **change)


def _meta(**change):
    def f(v):
        for k, g in change.items():
            setattr(v["meta"], k, g(getattr(v["meta"], k)))
        return v["meta"]

    return f


@pytest.mark.gpu
@pytest.mark.parametrize("call,names", [(_scan_call, ("dt", "a", "b", "c", "d", "z", "dt_bias", "state")), (_conv_call, ("w", "bias", "window"))])
def test_what_lies_elsewhere_or_is_too_short_is_refused(call, names):
    """Before anything is launched: tensors of the host, metadata of other types or for fewer sequences."""
    for name in names:
        with pytest.raises(ValueError):
            call("cuda", **{name: lambda v: v[name].cpu()})
    with pytest.raises(ValueError):
        call("cuda", out=lambda v: torch.zeros(4, 8))
    for change in (dict(query_start=lambda q: q.cpu()), dict(seq_lens=lambda q: q.long()), dict(state_slots=lambda q: q[:0]),
                   dict(query_start=lambda q: q[:1]), dict(query_start=lambda q: torch.stack([q, q], 1)[:, 0])):
        with pytest.raises(ValueError):
            call("cuda", meta=_meta(**change))


# ------------------------------------------------------------------------------------------------- graphs and streams
@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1] * 5, [6, 1, 30]])
def test_graphs_and_other_streams(lens):
    """Captured on one stream, replayed on new inputs: the same bits as eager calls one after another on a third."""
    gen = torch.Generator().manual_seed(21)
    C, N, K, T = 200, 16, 4, sum(lens)
    fixed = scan_inputs(gen, T, C, N, "f32", "f32", "f32", "bf16", True, True, True, 0, "cuda")
    x, w = rows(gen, T, C, torch.bfloat16, "cuda"), torch.randn(C, K, generator=gen).cuda()
    meta = step(lens, "cuda", fresh=())
    kept = [torch.randn(len(lens) + 2, K, C, generator=gen).cuda(), torch.randn(len(lens) + 2, C, N, generator=gen).cuda()]

    def call(window, state):
        u = ops.causal_conv(x, w, None, meta, window)
        return ops.selective_scan(**dict(fixed, u=u), meta=meta, state=state, act_dtype=torch.bfloat16)

    inputs = [(torch.randn(T, C, generator=gen).bfloat16().cuda(), torch.randn(T, C, generator=gen).cuda()) for _ in range(3)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    eager, mine = [], [k.clone() for k in kept]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for a, b in inputs:
            x.copy_(a)
            fixed["dt"].copy_(b)
            eager.append(call(*mine).clone())
    side.synchronize()
    held = [k.clone() for k in kept]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(*held)
    for a, k in zip(held, kept):
        a.copy_(k)
    for (a, b), want in zip(inputs, eager):
        x.copy_(a)
        fixed["dt"].copy_(b)
        graph.replay()
        assert torch.equal(y, want)
    assert all(torch.equal(a, b) for a, b in zip(held, mine))


@pytest.mark.gpu
def test_long_sequences_and_many():
    """Against the same kernel fed token by token, whose single steps the cases above hold to 64 bits."""
    gen = torch.Generator().manual_seed(22)
    C, N, K = 72, 16, 4
    lens = [3000] + [1, 2] * 150
    T = sum(lens)
    v = scan_inputs(gen, T, C, N, "f32", "f32", "f32", "f32", True, True, True, 0, "cuda")
    x, w = rows(gen, T, C, torch.bfloat16, "cuda"), torch.randn(C, K, generator=gen).cuda()
    meta = step(lens, "cuda")
    B = len(lens)
    win, state = torch.randn(B + 2, K, C, generator=gen).cuda(), torch.randn(B + 2, C, N, generator=gen).cuda()
    win1, state1 = win.clone(), state.clone()
    y, s = ops.causal_conv(x, w, None, meta, win), ops.selective_scan(**v, meta=meta, state=state)
    begin = [a - n for n, a in meta.host_lens]
    qs, y1, s1 = meta.query_start.tolist(), torch.empty_like(y), torch.empty_like(s)
    for j in range(max(lens)):
        on = [b for b in range(B) if lens[b] > j]
        take = torch.tensor([qs[b] + j for b in on], device="cuda")
        i32 = lambda q: torch.tensor(q, dtype=torch.int32, device="cuda")  # noqa: E731
        one = SimpleNamespace(query_start=i32(list(range(len(on) + 1))), seq_lens=i32([begin[b] + j + 1 for b in on]),
                              state_slots=meta.state_slots[torch.tensor(on, device="cuda")], max_query_len=1, host_lens=None)
        y1[take] = ops.causal_conv(x[take], w, None, one, win1)
        s1[take] = ops.selective_scan(**{k: m[take] if k in ("u", "dt", "b", "c", "z") else m for k, m in v.items()}, meta=one, state=state1)
    assert torch.equal(y, y1) and torch.equal(win, win1) and torch.equal(s, s1) and torch.equal(state, state1)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1, 1, 1], [4, 1, 2]])
def test_slots_outside_the_store_are_reported(lens):
    """Such a sequence's rows become zeros, nothing is written for it, the status word names its slot."""
    from oxidize_b200.ops import cuda as C

    gen = torch.Generator().manual_seed(23)
    meta = step(lens, "cuda", slots=(1, 77, 0))
    T = sum(lens)
    v = scan_inputs(gen, T, 40, 16, "f32", "f32", "f32", "f32", True, True, True, 0, "cuda")
    w, window, state = torch.randn(40, 4, generator=gen).cuda(), torch.randn(3, 4, 40, generator=gen).cuda(), torch.randn(3, 40, 16, generator=gen).cuda()
    kept = window[2].clone(), state[2].clone()
    C.status()
    y = ops.causal_conv(v["u"], w, None, meta, window)
    assert C.status()[:2] == (6 + 1, 77)
    s = ops.selective_scan(**v, meta=meta, state=state)
    assert C.status()[:2] == (6 + 1, 77)
    mine = slice(lens[0], lens[0] + lens[1])
    assert (y[mine] == 0).all() and (s[mine] == 0).all() and torch.equal(window[2], kept[0]) and torch.equal(state[2], kept[1])
