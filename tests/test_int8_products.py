"""Products on 8-bit integers (weights of type "I8") against statements in 64 bits.

The sums are whole numbers, so what the result may be off by is float32's rounding (2^-24 relative, half a step) of the sum, of the
products with the two scales and of the bias's sum, and then bfloat16's (2^-8)."""
import pytest
import torch

from oxidize_b200 import ops
from oxidize_b200.models.weights import LinearWeight, QTensor, fuse_rows, qtensor_from_dense
from oxidize_b200.ops import ref
from oxidize_b200.quant import torch_quant

HALF = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def tokens(x, device):
    """bfloat16 values in the type that the device's models run in."""
    return x.bfloat16().to(device) if device == "cuda" else x.bfloat16().float()


def weight(gen, n, k, device):
    w = torch.randn(n, k, generator=gen) * torch.exp(torch.randn(n, 1, generator=gen))
    q = qtensor_from_dense(w, "I8", device)
    assert q.data.dtype == torch.int8 and q.data.stride(0) % 16 == 0 and q.data.data_ptr() % 16 == 0
    return q


def codes64(x):
    """rint(127 x / max|x|) of every row, ties to even, in exact arithmetic on the values' fractions."""
    from fractions import Fraction

    out = torch.zeros(x.shape, dtype=torch.float64)
    for t, row in enumerate(x.double().cpu().tolist()):
        most = max(abs(v) for v in row)
        if most > 0:
            out[t] = torch.tensor([float(round(Fraction(v) * 127 / Fraction(most))) for v in row], dtype=torch.float64)
    return out


def product64(x, q, bias):
    """(y, bound of float32's roundings)."""
    xd, w = x.double(), q.data.double()
    most = xd.abs().amax(1, keepdim=True)
    codes = torch.round(xd * 127 / torch.where(most > 0, most, 1.0))
    y = (codes @ w.t()) * (most / 127) * q.scales.double()
    err = 4 * HALF * y.abs()  # the sum, the token's scale, two products
    if bias is not None:
        y = y + bias.double()
        err = err + HALF * (y.abs() + err)
    return y, err * (1 + 1e-6) + 1e-40


def check(x, q, bias, y):
    want, err = product64(x, q, bias)
    rounding = (torch.finfo(y.dtype).eps / 2) * (want.abs() + err)
    assert ((y.double() - want).abs() <= err + rounding).all()


SHAPES = [  # tokens, n, k
    (1, 1, 1), (1, 128, 128), (2, 130, 64), (1, 5000, 1111), (16, 256, 512), (17, 300, 200), (33, 128, 2000), (64, 1024, 4096),
    (65, 129, 127), (128, 96, 129), (129, 200, 384), (257, 384, 640), (300, 1000, 77), (513, 136, 1040), (7, 72, 16384), (3, 2000, 5000),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("T,n,k", SHAPES)
def test_product(T, n, k, with_bias, device):
    gen = torch.Generator().manual_seed(T + n + k)
    x = tokens(torch.randn(T, k, generator=gen) * torch.exp(2 * torch.randn(T, 1, generator=gen)), device)
    q = weight(gen, n, k, device)
    bias = torch.randn(n, generator=gen).to(device) if with_bias else None
    y = ops.linear(x, LinearWeight([q], bias))
    assert y.dtype == x.dtype and y.shape == (T, n)
    check(x, q, bias, y)


@pytest.mark.parametrize("device", DEVICES)
def test_codes_are_the_nearest_ones(device):
    """Values on and next to halves, the smallest and largest of the type, zeros: the codes of exact arithmetic."""
    gen = torch.Generator().manual_seed(4)
    k = 192
    x = torch.randn(64, k, generator=gen)
    x[1], x[2] = x[1] * 5e37, x[2] * 1e-38
    x[3] = 0
    x[4] = torch.arange(k) * 2.0 ** -133  # subnormal ones
    x[5] = 3.3e38 * torch.linspace(-1, 1, k)
    x[6, 1:], x[6, 0] = (torch.arange(k - 1) - 90) * 0.5, 127.0  # every half from -45 on
    x[7, 1:], x[7, 0] = (torch.arange(k - 1) - 90) * 0.25, 63.5
    x = x.bfloat16()
    x[8:] = (x[8:].float() * 2.0 ** torch.randint(-9, 9, (56, k), generator=gen)).bfloat16()
    x = tokens(x, device)
    # a product with the unit matrix gives the codes times the scale
    unit = QTensor("I8", torch_quant.int8_rows(torch.eye(k, dtype=torch.int8, device=device)), (k, k), torch.ones(k, device=device))
    y = ops.linear(x, LinearWeight([unit])).double().cpu()
    most = x.abs().amax(1).cpu()
    want = (codes64(x).float() * (most.float() / 127)[:, None]).to(x.dtype).double()
    assert torch.equal(y, want)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_are_not_finite_come_out_as_nan_alone(device):
    gen = torch.Generator().manual_seed(5)
    x = tokens(torch.randn(20, 96, generator=gen), device)
    q = weight(gen, 40, 96, device)
    clean = ops.linear(x, LinearWeight([q]))
    x[3, 7], x[11, 0], x[19, 95] = float("inf"), float("nan"), float("-inf")
    y = ops.linear(x, LinearWeight([q]))
    bad = torch.zeros(20, dtype=torch.bool)
    bad[[3, 11, 19]] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("device", DEVICES)
def test_largest_codes_and_longest_rows(device):
    """Sums up to 127 * 127 * 131072: within 32 bits."""
    k = 131072
    x = torch.ones(2, k)
    x[1, ::2] = -1
    x = tokens(x, device)
    q = QTensor("I8", torch.full((3, k), 127, dtype=torch.int8, device=device), (3, k), torch.ones(3, device=device))
    q.data[2] = -127
    y = ops.linear(x, LinearWeight([q]))
    check(x, q, None, y)
    assert y[0, 0] > 1.6e7 and y[0, 2] < -1.6e7 and (y[1] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_segments_beside_other_encodings(device):
    """q | k of one encoding and v of another: the same rows as each of them alone; segments of a kind fuse into one."""
    gen = torch.Generator().manual_seed(6)
    x = tokens(torch.randn(9, 64, generator=gen), device)
    a, b = weight(gen, 24, 64, device), weight(gen, 11, 64, device)
    v = qtensor_from_dense(torch.randn(16, 64, generator=gen), "BF16", device)
    bias = torch.randn(51, generator=gen).to(device)
    parts = fuse_rows([a, b, v])
    assert [p.qtype for p in parts] == ["I8", "BF16"] and parts[0].shape == (35, 64)
    y = ops.linear(x, LinearWeight(parts, bias))
    check(x, a, bias[:24], y[:, :24])
    check(x, b, bias[24:35], y[:, 24:35])
    assert torch.equal(y[:, 35:], ops.linear(x, LinearWeight([v], bias[35:])))
    assert torch.equal(ops.linear(x, LinearWeight([a, b], bias[:35])), y[:, :35])


def test_encoding_and_its_rows():
    gen = torch.Generator().manual_seed(7)
    w = torch.randn(10, 50, generator=gen)
    w[3] = 0
    w[4] *= 1e-40
    q = qtensor_from_dense(w, "I8")
    dense = ref.dequantize_weight(q)
    assert (q.scales[3] == 0) and (dense[3] == 0).all() and q.data.abs().max() == 127
    most = w.abs().amax(1)
    fine = [i for i in range(10) if i != 4]
    # half a code, and the roundings of the quotient, the scale and its product
    assert ((dense - w).abs() <= (most / 127 * (0.5 + 127 * 3 * HALF))[:, None])[fine].all()
    part = q.rows(2, 9)
    assert torch.equal(ref.dequantize_weight(part), dense[2:9]) and part.to("cpu").data.stride(0) % 16 == 0
    assert torch.equal(ref.dequantize_weight(q.to("cpu")), dense)


def test_random_weights_of_the_encoding():
    gen = torch.Generator().manual_seed(8)
    q = torch_quant.random_quantized(33, 70, "I8", "cpu", gen, 0.02)
    assert q.qtype == "I8" and q.shape == (33, 70) and 0.01 < ref.dequantize_weight(q).std() < 0.03


def _data(q):
    return q.data


@pytest.mark.gpu
@pytest.mark.parametrize("change", [
    lambda q: QTensor("I8", q.data.short(), q.shape, q.scales),  # another type
    lambda q: QTensor("I8", torch.zeros(40, 60, dtype=torch.int8, device="cuda"), (40, 60), q.scales),  # rows of 60 bytes
    lambda q: QTensor("I8", q.data, q.shape, q.scales.double()),
    lambda q: QTensor("I8", q.data[:, 16:48][:, 1:], (40, 31), q.scales),  # rows that start off a boundary
    lambda q: QTensor("I8", torch.zeros(40, 32, dtype=torch.int8, device="cuda"), (40, 32), q.scales),  # another width
    lambda q: QTensor("I8", torch.zeros(1, 131088, dtype=torch.int8, device="cuda"), (1, 131088), q.scales[:1])])
def test_what_the_kernel_does_not_read_is_refused(change):
    gen = torch.Generator().manual_seed(9)
    q = change(weight(gen, 40, 64, "cuda"))
    k = {60: 60, 31: 31, 131088: 131088}.get(q.shape[1], 64)
    with pytest.raises(ValueError):
        ops.linear(torch.zeros(3, k, dtype=torch.bfloat16, device="cuda"), LinearWeight([q]))


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,k", [(1, 640, 2048), (40, 512, 8192), (300, 256, 512)])
def test_graphs_other_streams_and_slices(T, n, k):
    """Captured and replayed on new inputs beside eager calls on another stream, into columns of a wider buffer: the same bits."""
    from oxidize_b200.ops import cuda as C

    gen = torch.Generator().manual_seed(10)
    q, bias = weight(gen, n, k, "cuda"), torch.randn(n, generator=gen).cuda()
    lw = LinearWeight([q], bias)
    inputs = [torch.randn(T, k, generator=gen).bfloat16().cuda() for _ in range(3)]
    want = [ops.linear(x, lw) for x in inputs]
    for x, y in zip(inputs, want):
        check(x, q, bias, y)
    x = inputs[0].clone()
    wide = torch.full((T + 2, n + 21), 3.0, dtype=torch.bfloat16, device="cuda")
    view = wide[1:-1, 5 : 5 + n]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = ops.linear(x, lw)
        C.linear(x, [q], bias, view)
    for a, b in zip(inputs, want):
        x.copy_(a)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = [ops.linear(v, lw) for v in inputs]
        torch.cuda.synchronize()
        assert torch.equal(y, b) and torch.equal(view, b) and all(torch.equal(o, v) for o, v in zip(other, want))
    assert (wide[0] == 3).all() and (wide[-1] == 3).all() and (wide[:, :5] == 3).all() and (wide[:, 5 + n :] == 3).all()
    assert C.status()[0] == 0


@pytest.mark.gpu
def test_no_tokens():
    gen = torch.Generator().manual_seed(11)
    assert ops.linear(torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda"), LinearWeight([weight(gen, 8, 64, "cuda")])).shape == (0, 8)


# ------------------------------------------------------------------------------------------------------- whole models
def _tiny_llama(path):
    from oxidize_b200.models.config import preset
    from oxidize_b200.utils.synth import synth_gguf

    synth_gguf(path, preset("tiny-llama", n_layers=2, vocab_size=300, hidden_size=128, n_heads=4, n_kv_heads=2, head_dim=64, ffn_size=192),
               "F32", seed=2, norm_jitter=0.1)
    return path


def _tiny_mamba(directory):
    T = pytest.importorskip("transformers")
    from oxidize_b200.formats.convert import convert_safetensors_to_gguf

    torch.manual_seed(0)
    model = T.MambaForCausalLM(T.MambaConfig(vocab_size=300, hidden_size=96, state_size=16, num_hidden_layers=2, conv_kernel=4, expand=2,
                                             time_step_rank=6))
    model.save_pretrained(str(directory / "hf"), safe_serialization=True)
    return convert_safetensors_to_gguf(str(directory / "hf"), str(directory / "m.gguf"), "F32")


def _llm(path, device, transcode="I8"):
    from oxidize_b200.engine.llm import LLM, EngineConfig

    return LLM.from_gguf(path, EngineConfig(max_model_len=128, max_num_seqs=4, num_kv_blocks=64, prefill_chunk_size=32, weight_transcode=transcode),
                         device=device)


def _far(a, b):
    return float((torch.as_tensor(a) - torch.as_tensor(b)).norm() / torch.as_tensor(b).norm())


@pytest.mark.parametrize("family", ["llama", "mamba"])
def test_projections_become_integers_while_loading(family, tmp_path):
    """Which ones do, and what that costs: with steps of 1/127 of a row's largest value (2.5 to 4 deviations) either side of a product is
    off by 0.6 to 0.9 percent of its size, which leaves room for ten products on the way within 5 percent (and twice that allowed)."""
    path = _tiny_llama(str(tmp_path / "m.gguf")) if family == "llama" else _tiny_mamba(tmp_path)
    plain, ints = _llm(path, "cpu", ""), _llm(path, "cpu", "i8")
    lw = ints.weights.layers[1]
    if family == "llama":
        assert [p.qtype for w in (lw.wqkv, lw.wo, lw.w_gate_up, lw.w_down) for p in w.parts] == ["I8"] * 4
    else:
        assert lw.ssm.in_proj.qtype == lw.ssm.out_proj.parts[0].qtype == "I8" and lw.ssm.x_proj.qtype == lw.ssm.dt_proj.qtype == "F32"
    assert ints.weights.embed.qtype == "F32" and (family == "mamba" or ints.weights.nbytes() < plain.weights.nbytes())
    prompt = [[5, 9, 20, 31, 200, 7]]
    assert 0 < _far(ints.next_token_logits(prompt), plain.next_token_logits(prompt)) < 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["llama", "mamba"])
def test_models_on_integers(family, tmp_path):
    """Prompts in portions, batches and single tokens on the device against the CPU's float32 path over the same integers: bfloat16
    activations (0.4 percent a rounding) move some codes by one."""
    from oxidize_b200.engine.sampler import SamplingParams

    path = _tiny_llama(str(tmp_path / "m.gguf")) if family == "llama" else _tiny_mamba(tmp_path)
    cpu, gpu = _llm(path, "cpu"), _llm(path, "cuda")
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(3, 300, (n,), generator=gen).tolist() for n in (5, 70, 1, 33)]
    for _ in range(2):
        a, b = cpu.next_token_logits(prompts), gpu.next_token_logits(prompts)
        assert _far(b, a) < 0.1
        prompts = [p + [int(torch.as_tensor(a)[i].argmax())] for i, p in enumerate(prompts)]
    out = gpu.generate(prompts, SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True))
    assert all(len(o.token_ids) == 8 for o in out)


def test_other_encodings_are_refused(tmp_path):
    from oxidize_b200.cli import main as cli

    path = _tiny_llama(str(tmp_path / "m.gguf"))
    with pytest.raises(ValueError):
        _llm(path, "cpu", "I4")
    with pytest.raises(SystemExit):
        cli.main(["run", path, "hi", "--int8", "--turboquant"])


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,k", [(1000, 5000, 300), (2049, 2300, 1000), (4096, 4096, 128), (777, 9000, 2050), (1500, 6001, 17), (257, 40000, 520)])
def test_many_tokens(T, n, k):
    """Many tiles, odd edges on all sides, twice in a row."""
    from oxidize_b200.ops import cuda as C

    gen = torch.Generator().manual_seed(T)
    q = weight(gen, n, k, "cuda")
    bias = torch.randn(n, generator=gen).cuda()
    for _ in range(2):
        x = torch.randn(T, k, generator=gen).bfloat16().cuda()
        check(x, q, bias, ops.linear(x, LinearWeight([q], bias)))
    assert C.status()[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 3, 5])
@pytest.mark.parametrize("k", [16, 40959, 40976, 512, 1023])
def test_few_tokens(T, k):
    """Both sides of where single tokens have a kernel of their own; a matrix that ends with its last value."""
    gen = torch.Generator().manual_seed(k)
    q = weight(gen, 70, k, "cuda")
    x = torch.randn(T, k, generator=gen).bfloat16().cuda()
    check(x, q, None, ops.linear(x, LinearWeight([q])))


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,k", [(2053, 6001, 130), (2304, 6016, 1040), (4100, 9216, 64)])
def test_last_waves(T, n, k):
    """Some more tiles than SMs, or twice as many: the last ones come in halves, one of which may have no rows at all."""
    from oxidize_b200.ops import cuda as C

    gen = torch.Generator().manual_seed(n)
    q = weight(gen, n, k, "cuda")
    bias = torch.randn(n, generator=gen).cuda()
    x = torch.randn(T, k, generator=gen).bfloat16().cuda()
    out = torch.full((T, n + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    check(x, q, bias, ops.linear(x, LinearWeight([q], bias)))
    ops.linear(x, LinearWeight([q], bias), out=out[:, :n])
    check(x, q, bias, out[:, :n])
    assert (out[:, n:] == 7).all() and C.status()[0] == 0


@pytest.mark.gpu
def test_what_lies_elsewhere_or_is_too_short_is_refused():
    """Before anything is launched; a bias of another type is converted."""
    gen = torch.Generator().manual_seed(10)
    q, x = weight(gen, 40, 64, "cuda"), torch.randn(3, 64, generator=gen).bfloat16().cuda()
    for bad in (QTensor("I8", q.data.cpu(), q.shape, q.scales), QTensor("I8", q.data, q.shape, q.scales.cpu()),
                QTensor("I8", q.data, q.shape, q.scales[:39]), QTensor("I8", q.data[:39], q.shape, q.scales),
                QTensor("I8", q.data, q.shape, q.scales[:1].expand(40))):
        with pytest.raises(ValueError):
            ops.linear(x, LinearWeight([bad]))
    with pytest.raises(ValueError):
        ops.linear(x, LinearWeight([q], torch.zeros(40)))
    bias = torch.randn(40, generator=gen).bfloat16().cuda()
    check(x, q, bias, ops.linear(x, LinearWeight([q], bias)))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 20, 50, 65, 100, 128])
@pytest.mark.parametrize("n,k", [(300, 4096), (100, 9000), (1025, 7300), (2600, 2100)])
def test_sums_in_shares(T, n, k):
    """Few weight tiles and long rows: several blocks share a tile's sums, each ends some of its tokens."""
    from oxidize_b200.ops import cuda as C

    gen = torch.Generator().manual_seed(T * n)
    q = weight(gen, n, k, "cuda")
    bias = torch.randn(n, generator=gen).cuda()
    x = torch.randn(T, k, generator=gen).bfloat16().cuda()
    y = ops.linear(x, LinearWeight([q], bias))
    check(x, q, bias, y)
    assert torch.equal(ops.linear(x, LinearWeight([q], bias)), y) and C.status()[0] == 0
