"""Steps of state-space layers that the tests of ``test_state_space.py`` do not make: metadata that contradicts itself, kernels that
only wide steps reach, values that are not finite, outputs over inputs.  Statements in 64 bits, bounds and tolerances are those."""
import pytest
import torch

from oxidize_b200 import ops
from test_state_space import DEVICES, TYPE, out_bound, scan64, scan_inputs, step


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("taps", [3, 4, 6])
@pytest.mark.parametrize("lens", [[1, 1, 1], [3, 5, 2]])
def test_lengths_below_the_rows_of_a_step(lens, taps, device):
    """A length that leaves a sequence's rows before position 0: refused on the CPU; on the device its rows become zeros, nothing is
    written for it, the status word has the length, and its neighbours are as without it."""
    gen = torch.Generator().manual_seed(31)
    C, N, T = 40, 16, sum(lens)
    v = scan_inputs(gen, T, C, N, "f32", "f32", "f32", "f32", True, True, True, 0, device)
    w = torch.randn(C, taps, generator=gen).to(device)
    # (slot 1 in the middle of the store: what lies ahead of its ring is slot 0's)
    window, state = torch.randn(3, taps, C, generator=gen).to(device), torch.randn(3, C, N, generator=gen).to(device)
    bad, none = step(lens, device, slots=(0, 1, 2)), step(lens, device, slots=(0, -1, 2))
    bad.seq_lens[1] = lens[1] - 1
    if device == "cpu":
        with pytest.raises(ValueError, match="length"):
            ops.causal_conv(v["u"], w, None, bad, window)
        with pytest.raises(ValueError, match="length"):
            ops.selective_scan(**v, meta=bad, state=state)
        return
    from oxidize_b200.ops import cuda as K

    window1, state1 = window.clone(), state.clone()
    K.status()
    y = ops.causal_conv(v["u"], w, None, bad, window)
    assert K.status()[:2] == (8, lens[1] - 1)
    s = ops.selective_scan(**v, meta=bad, state=state)
    assert K.status()[:2] == (8, lens[1] - 1)
    y1, s1 = ops.causal_conv(v["u"], w, None, none, window1), ops.selective_scan(**v, meta=none, state=state1)
    assert K.status()[0] == 0
    assert torch.equal(y, y1) and torch.equal(s, s1) and torch.equal(window, window1) and torch.equal(state, state1)


@pytest.mark.parametrize("apart", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 8])
def test_rows_far_apart(apart):
    """The kernels take the distance of rows as a 32-bit number: rows further apart are copied, such an output is refused; one row
    alone has no next one.  (Of the bindings, which launch nothing here: tensors without storage.)"""
    from oxidize_b200.ops import cuda_ssm

    far = torch.empty_strided((2, 8), (apart, 1), device="meta")
    x, (_, ld, code) = cuda_ssm._rows(far, "x")
    assert x.shape == (2, 8) and code == 0 and ld == (apart if apart < 2 ** 31 else 8)
    one, _ = cuda_ssm._rows(far[:1], "x")
    assert one.stride() == (apart, 1)
    if apart < 2 ** 31:
        assert cuda_ssm._out(far, 2, 8, torch.float32, far) is far
    else:
        with pytest.raises(ValueError, match="apart"):
            cuda_ssm._out(far, 2, 8, torch.float32, far)
    assert cuda_ssm._out(far[:1], 1, 8, torch.float32, far) is not None


def test_steps_of_a_model_are_freed_with_their_last_name(tmp_path, monkeypatch):
    """Without Python's collector of cycles: a step's tensors go when the step does."""
    import gc
    import weakref

    from test_int8_products import _llm, _tiny_mamba

    llm = _llm(_tiny_mamba(tmp_path), "cpu", "")
    seen, slots_of = [], llm.model._ssm_step

    def watched(meta, kv, first_layer):
        out = slots_of(meta, kv, first_layer)
        seen.extend((weakref.ref(meta), weakref.ref(out), weakref.ref(out.state_slots)))
        return out

    monkeypatch.setattr(llm.model, "_ssm_step", watched)
    gc.collect()
    gc.disable()
    try:
        llm.next_token_logits([[5, 9, 20], [31]])
        assert len(seen) >= 6 and all(r() is None for r in seen)
    finally:
        gc.enable()


def _mamba_with_states(directory, states):
    T = pytest.importorskip("transformers")
    from oxidize_b200.formats.convert import convert_safetensors_to_gguf

    torch.manual_seed(0)
    model = T.MambaForCausalLM(T.MambaConfig(vocab_size=300, hidden_size=64, state_size=states, num_hidden_layers=2, conv_kernel=4, expand=2,
                                             time_step_rank=4))
    model.save_pretrained(str(directory / "hf"), safe_serialization=True)
    return convert_safetensors_to_gguf(str(directory / "hf"), str(directory / "m.gguf"), "F32")


@pytest.mark.gpu
@pytest.mark.parametrize("states", [128, 129, 200])
def test_models_with_many_states(states, tmp_path):
    """On either side of what the scan's kernel takes, against the CPU (the tolerance of the other engine tests: bfloat16 projections)."""
    from test_int8_products import _far, _llm

    path = _mamba_with_states(tmp_path, states)
    cpu, gpu = _llm(path, "cpu", ""), _llm(path, "cuda", "")
    prompts = [[5, 9, 20, 31, 200, 7], [17]]
    for _ in range(2):
        a, b = cpu.next_token_logits(prompts), gpu.next_token_logits(prompts)
        assert _far(b, a) < 0.1
        prompts = [p + [int(torch.as_tensor(a)[i].argmax())] for i, p in enumerate(prompts)]


# lens, channels: single rows; 16 and 8 lanes and one lane to a channel (with 148 SMs, see lanes())
STEPS = {"single rows": ([1] * 9, 40), "16 lanes": ([70, 3, 17], 40), "8 lanes": ([37, 70], 1801), "one lane": ([70, 70, 70, 64, 33, 70, 1, 70], 2726)}


def lanes(lens, C):
    """Lanes to a channel of up to 16 states that the device's kernel takes, of its rule on the channels that run at a time."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    channels = C * -(-sum(lens) // max(lens))
    return 16 if channels < 12 * sms else 8 if channels < 110 * sms else 1


def check_kernel(kind, lens, C):
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert kind == "single rows" or lanes(lens, C) == {"16 lanes": 16, "8 lanes": 8, "one lane": 1}[kind]


# (the CPU has one statement for all of them)
@pytest.mark.parametrize("kind,device", [(k, "cpu") for k, (_, C) in STEPS.items() if C < 100] + [pytest.param(k, "cuda", marks=pytest.mark.gpu) for k in STEPS])
@pytest.mark.parametrize("N,gate,types", [(1, False, "f32"), (5, True, "f32"), (8, False, "bf16"), (11, False, "f32"), (13, True, "bf16"), (16, True, "f32"), (24, False, "f32"),
                                          (100, True, "f32")])
def test_steps_that_are_not_finite(N, gate, types, kind, device):
    """Inputs and steps that are infinite or NaN: infinities stay infinities, whatever the number of states is padded to."""
    lens, C = STEPS[kind]
    if device == "cuda":
        check_kernel(kind, lens, C)
    gen = torch.Generator().manual_seed(51)
    meta = step(lens, device, slots=range(len(lens)))
    v = scan_inputs(gen, sum(lens), C, N, types, types, "f32", "f32", gate, True, True, 0, device)
    v["b"], v["c"] = v["b"].abs(), v["c"].abs()  # (sums of infinities of one sign)
    end = int(meta.query_start[1])
    strange = {(end - 1, 3): ("u", float("inf")), (0, 7): ("u", float("-inf")), (end // 2, C - 1): ("dt", float("inf")), (end, 5): ("u", float("nan")),
               (sum(lens) - 1, 0): ("u", float("inf"))}
    for (t, c), (name, value) in strange.items():
        v[name][t, c] = value
    state = torch.randn(len(lens) + 2, C, N, generator=gen).to(device)
    want, err, after, after_err = scan64(**v, meta=meta, state=state)
    y = ops.selective_scan(**v, meta=meta, state=state)
    assert torch.isinf(want).any() and torch.isnan(want).any()
    for got, exact, bound in ((y.double(), want, err), (state.double(), after, after_err)):
        fine = torch.isfinite(exact)
        assert ((got - exact).abs() <= bound)[fine].all()
        assert torch.equal(torch.isnan(got), torch.isnan(exact)) and torch.equal(got[torch.isinf(exact)], exact[torch.isinf(exact)])


def test_what_shares_memory_with_an_output():
    """Against the sets of bytes themselves."""
    from oxidize_b200.ops import cuda_ssm

    store = torch.zeros(400)
    gen = torch.Generator().manual_seed(61)
    pick = lambda n: int(torch.randint(0, n, (1,), generator=gen))  # noqa: E731

    def matrix(ld):
        v = store if pick(3) else store.view(torch.bfloat16)
        return v.as_strided((T, 1 + pick(9)), (ld * (4 // v.element_size()), 1), pick(90))

    def held(v):
        rows = range(v.shape[0])
        return {v.data_ptr() + (r * v.stride(0) + c) * v.element_size() + b for r in rows for c in range(v.shape[1]) for b in range(v.element_size())}

    seen = set()
    for _ in range(2000):
        T = 1 + pick(5)
        ld = 9 + pick(12)
        v, out = matrix(ld), matrix(ld if pick(4) else 9 + pick(12))
        shared = bool(held(v) & held(out))
        copied = cuda_ssm._apart(v, out).data_ptr() != v.data_ptr()
        # rows of other lengths count as sharing as soon as the matrices interleave
        assert copied == shared if v.stride(0) * v.element_size() == out.stride(0) * out.element_size() else copied >= shared
        seen.add((shared, copied))
    assert {(True, True), (False, False)} <= seen
    assert cuda_ssm._apart(None, store[None]) is None and cuda_ssm._apart(store[None], None) is not None


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [[1] * 6, [300, 1, 64]])
def test_outputs_over_inputs(lens, device):
    """Over the input itself, or one row further: as into memory of its own."""
    gen = torch.Generator().manual_seed(62)
    C, N, T = 72, 11, sum(lens)
    meta = step(lens, device)
    w = torch.randn(C, 4, generator=gen).to(device)
    v = scan_inputs(gen, T, C, N, "f32", "f32", "f32", "f32", True, True, True, 0, device)
    v["u"][T // 2, 3] = float("inf")
    window, state = torch.randn(len(lens) + 2, 4, C, generator=gen).to(device), torch.randn(len(lens) + 2, C, N, generator=gen).to(device)
    conv = lambda x, out: ops.causal_conv(x, w, None, meta, window.clone(), out=out)  # noqa: E731
    scan = lambda name, x, out: ops.selective_scan(**dict(v, **{name: x}), meta=meta, state=state.clone(), out=out)  # noqa: E731
    same = lambda a, b: torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))  # noqa: E731
    for name, call in [("u", lambda x, out: conv(x, out))] + [(n, lambda x, out, n=n: scan(n, x, out)) for n in ("u", "dt", "z")]:
        # over it, a row further, and columns beside it (the same strides either way: the CPU takes vector and scalar forms of its functions
        # by them)
        for ahead, beside in ((0, 0), (C, 0), (0, C)):
            room = torch.zeros((T + 1) * (C + beside), device=device)
            x, out = (room.as_strided((T, C), (C + beside, 1), at) for at in (0, ahead + beside))
            x.copy_(v[name])
            want = call(x, None)
            got = call(x, out)
            assert got is out and same(got, want)


@pytest.mark.gpu
def test_more_rows_than_the_step_says():
    """max_query_len 1 (which metadata has where nobody sets it) and a sequence of three rows: reported, zeros, its state as it was; the
    others as ever.  The convolution does not go by it."""
    from oxidize_b200.ops import cuda as K

    gen = torch.Generator().manual_seed(71)
    C, N, lens = 200, 16, [1, 3, 1, 0, 1]
    meta = step(lens, "cuda", slots=(0, 1, 2, 3, 4), fresh=())
    v = scan_inputs(gen, 6, C, N, "f32", "f32", "f32", "f32", True, True, True, 0, "cuda")
    w, window, state = torch.randn(C, 4, generator=gen).cuda(), torch.randn(7, 4, C, generator=gen).cuda(), torch.randn(7, C, N, generator=gen).cuda()
    window1, state1 = window.clone(), state.clone()
    y, s = ops.causal_conv(v["u"], w, None, meta, window), ops.selective_scan(**v, meta=meta, state=state)
    kept = state1.clone()
    meta.max_query_len = 1
    K.status()
    assert torch.equal(ops.causal_conv(v["u"], w, None, meta, window1), y) and torch.equal(window, window1) and K.status()[0] == 0
    s1 = ops.selective_scan(**v, meta=meta, state=state1, out=torch.full_like(s, 7.0))
    assert K.status()[:2] == (8, 3)
    assert (s1[1:4] == 0).all() and torch.equal(s1[[0, 4, 5]], s[[0, 4, 5]])
    assert torch.equal(state1[1], kept[1]) and torch.equal(state1[[0, 2, 3, 4, 5, 6]], state[[0, 2, 3, 4, 5, 6]])


# Lengths off the tiles' multiples (8 and 32 rows), with none and with one row; channels off 32
WIDE = [70, 64, 0, 33, 70, 1, 61, 70, 70, 58, 9]


@pytest.mark.gpu
@pytest.mark.parametrize("N,C,tu,tbc,tout,gate", [(16, 2726, "f32", "f32", "bf16", True), (16, 2726, "bf16", "bf16", "f32", True), (16, 5121, "bf16", "f32", "bf16", False),
                                                  (11, 2726, "f32", "bf16", "f32", True), (12, 2752, "bf16", "f32", "f32", False), (8, 2726, "f32", "f32", "f32", True),
                                                  (5, 2735, "bf16", "bf16", "bf16", False), (8, 2752, "bf16", "bf16", "f32", False), (3, 2726, "f32", "f32", "bf16", True)])
def test_scan_with_a_lane_to_a_channel(N, C, tu, tbc, tout, gate):
    """Wide steps of prompts, one of which has no slot and one no rows."""
    gen = torch.Generator().manual_seed(81)
    check_kernel("one lane", WIDE, C)
    meta = step(WIDE, "cuda", no_slot=(4,))
    T = sum(WIDE)
    v = scan_inputs(gen, T + 2, C, N, tu, tu, tbc, tout, gate, True, True, 5, "cuda")
    state = torch.randn(len(WIDE) + 2, C, N, generator=gen).cuda()
    want, err, after, after_err = scan64(**v, meta=meta, state=state)
    out = torch.full((T + 2, C + 3), 7.0, dtype=TYPE[tout], device="cuda")
    y = ops.selective_scan(**v, meta=meta, state=state, act_dtype=TYPE[tout], out=out[:, 2 : 2 + C])[:T]
    assert ((y.double() - want[:T]).abs() <= out_bound(want, err, TYPE[tout])[:T]).all()
    assert ((state.double() - after).abs() <= after_err).all()
    assert (out[T:] == 7).all() and (out[:, :2] == 7).all() and (out[:, 2 + C :] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N,C", [(24, 1777), (32, 2001), (20, 6003)])
def test_scan_of_more_states_on_eight_lanes(N, C):
    gen = torch.Generator().manual_seed(82)
    lens = [70, 37, 1, 70]
    assert torch.cuda.get_device_properties(0).multi_processor_count != 148 or lanes(lens, C) <= 8
    meta = step(lens, "cuda")
    v = scan_inputs(gen, sum(lens), C, N, "f32", "f32", "f32", "f32", True, True, True, 3, "cuda")
    state = torch.randn(len(lens) + 2, C, N, generator=gen).cuda()
    want, err, after, after_err = scan64(**v, meta=meta, state=state)
    y = ops.selective_scan(**v, meta=meta, state=state)
    assert ((y.double() - want).abs() <= err).all() and ((state.double() - after).abs() <= after_err).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [16, 11, 8, 24])
def test_neighbours_that_change_the_kernel_leave_the_bits(N):
    """A sequence alone (8 lanes to a channel), in single rows, and beside others that bring a lane to a channel."""
    gen = torch.Generator().manual_seed(83)
    C, n = 2726, 70
    check_kernel("one lane", WIDE, C)
    check_kernel("8 lanes", [n], C)
    v = scan_inputs(gen, sum(WIDE), C, N, "f32", "f32", "f32", "f32", True, True, True, 0, "cuda")
    first = torch.randn(1, C, N, generator=gen).cuda()
    take = lambda rows: {k: m[rows] if k in ("u", "dt", "b", "c", "z") else m for k, m in v.items()}  # noqa: E731
    many = torch.randn(len(WIDE), C, N, generator=gen).cuda()
    many[0] = first[0]
    alone, rows = first.clone(), first.clone()

    def meta(lens, before, slots):
        m = step(lens, "cuda", slots=slots)
        m.seq_lens.copy_(torch.tensor([before + k for k in lens]))
        return m

    y = ops.selective_scan(**v, meta=meta(WIDE, 6, range(len(WIDE))), state=many)[:n]
    assert torch.equal(ops.selective_scan(**take(slice(0, n)), meta=meta([n], 6, (0,)), state=alone), y) and torch.equal(alone[0], many[0])
    for t in range(n):
        assert torch.equal(ops.selective_scan(**take(slice(t, t + 1)), meta=meta([1], 6 + t, (0,)), state=rows), y[t : t + 1])
    assert torch.equal(rows[0], many[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [[1, 1, 1], [3]])
def test_outputs_whose_rows_share_memory_are_refused(lens, device):
    """Also over an input of that kind; a row alone shares with no other."""
    gen = torch.Generator().manual_seed(91)
    C, meta = 8, step(lens, device)
    w, window, state = torch.zeros(C, 4, device=device), torch.zeros(5, 4, C, device=device), torch.zeros(5, C, 16, device=device)
    v = scan_inputs(gen, 3, C, 16, "f32", "f32", "f32", "f32", True, True, True, 0, device)
    room = torch.zeros(64, device=device)
    for apart in (0, 7):
        out = room.as_strided((3, C), (apart, 1))
        for x in (v["u"], out):
            with pytest.raises(ValueError, match="share"):
                ops.causal_conv(x, w, None, meta, window, out=out)
            with pytest.raises(ValueError, match="share"):
                ops.selective_scan(**dict(v, u=x), meta=meta, state=state, out=out)
    one = step([1], device)
    ops.causal_conv(v["u"][:1], w, None, one, window, out=room.as_strided((1, C), (0, 1)))
