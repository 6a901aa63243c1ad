"""Operators of state-space models and of 8-bit integer products: what is measured, on which inputs, and their plain form.

A case is one call as a serving process makes it: the short causal convolution of a step's rows, the selective scan over them, or a
projection whose weights are 8-bit integers with a scale per output channel and whose activations get a scale per token.  A step
feeds ragged sequences (``rows_lo`` .. ``rows_hi`` rows each, some of which go on from earlier positions); sizes are those of
state-space decoders (inner widths of 512 to 8192, 16 states, 4 taps) and of this repository's dense presets.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _conv(name, seqs, rows, width, taps, x, out, act="silu"):
    return {"name": name, "op": "conv", "seqs": seqs, "rows_lo": rows[0], "rows_hi": rows[1], "width": width, "taps": taps, "in": x, "out": out,
            "act": act}


def _scan(name, seqs, rows, width, states, x, out, gate=True):
    return {"name": name, "op": "scan", "seqs": seqs, "rows_lo": rows[0], "rows_hi": rows[1], "width": width, "states": states, "in": x, "out": out,
            "gate": gate}


def _int8(name, tokens, n, k, bias=False):
    return {"name": name, "op": "int8", "tokens": tokens, "n": n, "k": k, "bias": bias}


def listed():
    return [
        # one user's next token: a launch and a latency
        _conv("conv step 1", 1, (1, 1), 2048, 4, "bf16", "f32"),
        # a full batch of decoding sequences
        _conv("conv step 256", 256, (1, 1), 5120, 4, "bf16", "f32"),
        # the scheduler's step of prompts: ragged, some of them going on from an earlier portion
        _conv("conv prompts 7", 7, (300, 1900), 4096, 4, "bf16", "f32"),
        # a long document through a model that runs in float32, of an odd width and without an activation
        _conv("conv long odd f32", 1, (16384, 16384), 2051, 3, "f32", "f32", act="none"),
        _scan("scan step 1", 1, (1, 1), 2048, 16, "f32", "bf16"),
        _scan("scan step 256", 256, (1, 1), 5120, 16, "f32", "bf16"),
        # one prompt of a small model: few channels for the machine's width
        _scan("scan prompt 2048", 1, (2048, 2048), 1536, 16, "f32", "bf16"),
        # the scheduler's step of prompts
        _scan("scan prompts 9", 9, (200, 1650), 5120, 16, "bf16", "bf16"),
        # odd widths, float32 throughout, without a gate
        _scan("scan odd f32", 3, (501, 1001), 1001, 11, "f32", "f32", gate=False),
        # a wide projection for one token: the weights' bytes
        _int8("int8 1 token", 1, 10240, 2560),
        # the gate and up projection of the benchmark's large model for its 64 sequences
        _int8("int8 64 tokens", 64, 57344, 8192),
        # a portion of prompts: the tensor cores' rate
        _int8("int8 4096 tokens", 4096, 14336, 4096, bias=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("conv", "scan", "int8"))
    if op == "int8":
        tokens = log_int(1, 4096)
        n, k = log_int(64, 16384), log_int(64, 16384)
        if rng.random() < 0.6:
            n, k = max(64, n // 128 * 128), max(64, k // 64 * 64)
        k = min(k, max(64, int(2.4e11 / (tokens * n))))
        c = _int8("", tokens, n, k, bias=rng.random() < 0.5)
    else:
        width = log_int(256, 8192)
        if rng.random() < 0.6:
            width = width // 64 * 64
        if rng.random() < 0.4:
            seqs, rows = log_int(1, 256), (1, 1)
        else:
            total = log_int(64, max(64, int((3.0e7 if op == "conv" else 2.5e7) / width)))
            seqs = rng.randint(1, min(12, total))
            hi = max(1, total // seqs)
            rows = (rng.randint(1, hi), hi)
        if op == "conv":
            c = _conv("", seqs, rows, width, rng.choice((2, 3, 4, 4, 4)), rng.choice(("bf16", "bf16", "f32")), rng.choice(("f32", "f32", "bf16")),
                      rng.choice(("silu", "silu", "none")))
        else:
            c = _scan("", seqs, rows, width, rng.choice((8, 16, 16, 16, rng.randint(1, 24))), rng.choice(("f32", "f32", "bf16")),
                      rng.choice(("bf16", "bf16", "f32")), rng.random() < 0.8)
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------------------------- inputs
def _lens(c):
    """Rows that each sequence feeds: from rows_lo to rows_hi, all over the range (one sequence: rows_hi)."""
    lo, hi, n = c["rows_lo"], c["rows_hi"], c["seqs"]
    return [hi if i == 0 else lo + round((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


def _step(c, gen):
    """What the engine says of a step: where each sequence's rows are, its length with them, the slot of its state."""
    lens = _lens(c)
    decode = c["rows_hi"] == 1
    # prompts: every second sequence is at its start; decoding sequences are somewhere
    before = [int(torch.randint(1, 5000, (1,), generator=gen)) if decode or i % 2 else 0 for i in range(len(lens))]
    start = [0]
    for n in lens:
        start.append(start[-1] + n)
    slots = torch.randperm(len(lens) + 1, generator=gen)[: len(lens)]
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).to(DEV)  # noqa: E731
    return SimpleNamespace(query_start=i32(start), seq_lens=i32([b + n for b, n in zip(before, lens)]), state_slots=i32(slots), max_query_len=max(lens),
                           host_lens=[(n, b + n) for b, n in zip(before, lens)], extra={})


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.empty(*shape, device=DEV).normal_(0.0, std, generator=gen)

    if case["op"] == "int8":
        t, n, k = case["tokens"], case["n"], case["k"]
        x = normal(t, k)
        x[:, ::61] *= 8.0  # a few channels are large, as a decoder's are
        if t > 8:
            x[t // 2] = 0.0  # a padding row
        scales = torch.empty(n, device=DEV)
        # rows of 16-byte multiples, as the loader lays them out
        codes = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device=DEV)[:, :k]
        for r in range(0, n, 8192):
            w = normal(min(8192, n - r), k, std=0.02)
            scales[r : r + 8192] = w.abs().amax(1) / 127
            codes[r : r + 8192] = torch.round(w / scales[r : r + 8192, None]).to(torch.int8)
        return {"case": case, "x": x.bfloat16(), "codes": codes, "scales": scales, "bias": normal(n) if case["bias"] else None}
    meta = _step(case, host)
    T, W, slots = sum(_lens(case)), case["width"], case["seqs"] + 1
    kind = TYPES[case["in"]]
    if case["op"] == "conv":
        K = case["taps"]
        # the left half of an input projection's rows
        return {"case": case, "meta": meta, "x": normal(T, 2 * W).to(kind)[:, :W], "w": normal(W, K, std=K ** -0.5), "bias": normal(W, std=0.1),
                "window": normal(slots, K, W).to(kind).float()}
    N = case["states"]
    par = normal(T, 2 * N)  # B and C are neighbouring columns of one projection's rows
    step = torch.exp(torch.empty(W, device=DEV).uniform_(math.log(1e-3), math.log(1e-1), generator=gen))
    a = -torch.arange(1, N + 1, device=DEV, dtype=torch.float32) * torch.exp(normal(W, N, std=0.1))
    u = torch.nn.functional.silu(normal(T, W))
    return {"case": case, "meta": meta, "u": u.to(kind), "dt": normal(T, W, std=0.7).to(kind), "b": par[:, :N], "c": par[:, N:],
            # the gate is the right half of the input projection's rows
            "z": normal(T, 2 * W).to(torch.bfloat16 if case["out"] == "bf16" else torch.float32)[:, W:] if case["gate"] else None, "a": a.contiguous(),
            "d": 1 + normal(W, std=0.1), "dt_bias": step + torch.log(-torch.expm1(-step)), "state": normal(slots, W, N, std=0.3)}


# -------------------------------------------------------------------------------------------------------- plain form
def _rows(meta, T):
    """(sequence of each row, its place among the sequence's rows), and the sequences' first rows and lengths."""
    first, upto = meta.query_start[:-1].long(), meta.query_start[1:].long()
    at = torch.arange(T, device=DEV)
    seq = torch.searchsorted(upto, at, right=True)
    return seq, at - first[seq], first, upto - first


def _silu(x):
    return x / (1 + torch.exp(-x))


def _plain_conv(s):
    c, meta, window = s["case"], s["meta"], s["window"]
    x, w, K = s["x"].float(), s["w"], c["taps"]
    T = x.shape[0]
    seq, place, first, lens = _rows(meta, T)
    slot, before = meta.state_slots.long(), meta.seq_lens.long() - lens
    back = torch.arange(K - 1, -1, -1, device=DEV)  # tap i is K - 1 - i rows back

    def inputs(row, b, j, pos):
        """The inputs 0 .. K - 1 rows before places j of sequences b ([.., 1] each): a row of this step, of the window, or nothing."""
        here, old = x[(row - back).clamp_min(0)], window[slot[b], (pos - back) % K]
        return torch.where((j >= back)[..., None], here, old) * (pos >= back)[..., None]

    every = inputs(torch.arange(T, device=DEV)[:, None], seq[:, None], place[:, None], (before[seq] + place)[:, None])  # [T, K, width]
    y = (every * w.t()).sum(1) + s["bias"]
    # the last rows of a sequence, K at most, stay for its next step
    row, pos = (first + lens - 1)[:, None] - back, ((before + lens - 1)[:, None] - back) % K
    window[slot[:, None], pos] = torch.where((row >= first[:, None])[..., None], x[row.clamp_min(0)], window[slot[:, None], pos])
    return {"y": (_silu(y) if c["act"] == "silu" else y).to(TYPES[c["out"]]), "window": window}


def _plain_scan(s):
    c, meta, state = s["case"], s["meta"], s["state"]
    u, z = s["u"].float(), s["z"]
    T = u.shape[0]
    seq, place, first, lens = _rows(meta, T)
    slot = meta.state_slots.long()
    dt = s["dt"].float() + s["dt_bias"]
    dt = torch.where(dt > 20, dt, torch.log1p(torch.exp(dt.clamp_max(20))))
    keep = torch.exp(dt[:, :, None] * s["a"])
    h = (dt * u)[:, :, None] * s["b"][:, None, :]
    # a sequence starts from its state, or from nothing at position 0, and from no row before it
    h[first] += keep[first] * state[slot] * (meta.seq_lens.long() > lens)[:, None, None]
    keep[first] = 0
    # h_t = keep_t h_{t-1} + h_t: spans of twice the length each time
    span = 1
    while span < meta.max_query_len:
        h = torch.cat([h[:span], h[span:] + keep[span:] * h[:-span]])
        keep = torch.cat([keep[:span], keep[span:] * keep[:-span]])
        span *= 2
    y = (h * s["c"][:, None, :]).sum(-1) + s["d"] * u
    if z is not None:
        y = y * _silu(z.float())
    state[slot] = h[first + lens - 1]
    return {"y": y.to(TYPES[c["out"]]), "state": state}


def _plain_int8(s):
    x = s["x"].float()
    most = x.abs().amax(1, keepdim=True)
    # (64 bits: codes next to a border)
    codes = torch.round(x.double() * 127 / most.double().clamp_min(1e-300)).float()
    y = (codes @ s["codes"].float().t()) * (most / 127) * s["scales"]
    return (y if s["bias"] is None else y + s["bias"]).bfloat16()


def run(state):
    c = state["case"]
    if not own:
        return {"conv": _plain_conv, "scan": _plain_scan, "int8": _plain_int8}[c["op"]](state)
    from oxidize_b200 import ops

    s = state
    if c["op"] == "conv":
        y = ops.causal_conv(s["x"], s["w"], s["bias"], s["meta"], s["window"], act=c["act"], act_dtype=TYPES[c["out"]])
        return {"y": y, "window": s["window"]}
    if c["op"] == "scan":
        y = ops.selective_scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["d"], s["z"], s["dt_bias"], s["meta"], s["state"], act_dtype=TYPES[c["out"]])
        return {"y": y, "state": s["state"]}
    from oxidize_b200.models.weights import LinearWeight, QTensor

    return ops.linear(s["x"], LinearWeight([QTensor("I8", s["codes"], (c["n"], c["k"]), s["scales"])], s["bias"]))


# -------------------------------------------------------------------------------------------------- 64-bit definition
def _padded(rows, lens):
    """[T, ...] as [sequences, longest, ...] in 64 bits."""
    return torch.nn.utils.rnn.pad_sequence(list(rows.double().split(lens)), batch_first=True)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "int8":
        x = s["x"].double()
        most = x.abs().max(dim=1).values
        codes = torch.where(most[:, None] > 0, x / most[:, None].clamp_min(1e-300) * 127, 0 * x)
        near = (codes * 2).round() / 2  # halves that the quotient's rounding moved
        codes = torch.where((codes - near).abs() < 1e-10, near, codes).round()
        y = torch.einsum("tk,nk->tn", codes, s["codes"].double()) * torch.outer(most / 127, s["scales"].double())
        return y if s["bias"] is None else y + s["bias"].double()
    meta, lens, W = s["meta"], _lens(case), case["width"]
    before = [n - m for m, n in meta.host_lens]
    slots = meta.state_slots.tolist()
    mask = torch.arange(max(lens), device=DEV) < torch.tensor(lens, device=DEV)[:, None]
    if case["op"] == "conv":
        K, window = case["taps"], s["window"].double()
        parts, after, ys = list(s["x"].double().split(lens)), window.clone(), []
        for b, x in enumerate(parts):
            old = torch.stack([window[slots[b], p % K] if p >= 0 else torch.zeros(W, dtype=torch.float64, device=DEV)
                               for p in range(before[b] - K + 1, before[b])])
            full = torch.cat([old, x])
            ys.append(torch.nn.functional.conv1d(full.t()[None], s["w"].double()[:, None], s["bias"].double(), groups=W)[0].t())
            for i in range(max(0, len(x) - K), len(x)):
                after[slots[b], (before[b] + i) % K] = x[i]
        y = torch.cat(ys)
        return {"y": y * torch.sigmoid(y) if case["act"] == "silu" else y, "window": after}
    u, dt, bm, cm = (_padded(s[k], lens) for k in ("u", "dt", "b", "c"))
    dt = torch.logaddexp(dt + s["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device=DEV))
    a, fresh = s["a"].double(), torch.tensor([p == 0 for p in before], device=DEV)
    h = s["state"][slots].double().masked_fill(fresh[:, None, None], 0.0)
    y = torch.zeros_like(u)
    for t in range(max(lens)):
        new = h * torch.exp(dt[:, t, :, None] * a) + torch.einsum("bw,bn->bwn", dt[:, t] * u[:, t], bm[:, t])
        h = torch.where(mask[:, t, None, None], new, h)
        y[:, t] = torch.einsum("bwn,bn->bw", h, cm[:, t])
    y = (y + s["d"].double() * u)[mask]
    if s["z"] is not None:
        y = y * s["z"].double() * torch.sigmoid(s["z"].double())
    state = s["state"].double()
    state[slots] = h
    return {"y": y, "state": state}


def work(case):
    size = {"bf16": 2, "f32": 4}
    if case["op"] == "int8":
        t, n, k = case["tokens"], case["n"], case["k"]
        return {"bytes": 2 * t * k + n * k + 4 * n + 2 * t * n, "flops": 2 * t * n * k}
    lens, W = _lens(case), case["width"]
    T, B, x, y = sum(lens), len(lens), size[case["in"]], size[case["out"]]
    if case["op"] == "conv":
        K = case["taps"]
        rows = sum(min(n, K) for n in lens)  # of the window, written; as many or fewer are read
        return {"bytes": T * W * (x + y) + 4 * W * (rows + B * (K - 1)) + 4 * W * (K + 1), "flops": 2 * K * T * W}
    N = case["states"]
    gate = (2 if case["out"] == "bf16" else 4) if case["gate"] else 0
    # per state: the exponent, its exponential, the input's share, two fused steps of two operations each
    return {"bytes": T * W * (2 * x + y + gate) + 8 * T * N + 8 * B * W * N + 4 * W * (N + 2), "flops": 7 * T * W * N}
