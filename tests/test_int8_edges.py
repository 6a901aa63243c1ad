"""Calls of products on 8-bit integers that ``test_int8_products.py`` does not make.  Its statement in 64 bits and its bounds."""
import pytest
import torch

from oxidize_b200 import ops
from oxidize_b200.models.weights import LinearWeight, QTensor, qtensor_from_dense
from oxidize_b200.quant import torch_quant
from test_int8_products import DEVICES, check, tokens, weight


def far(n, k, apart, dtype):
    return torch.empty_strided((n, k), (apart, 1), dtype=dtype, device="meta")


@pytest.mark.parametrize("change", [
    dict(bias=torch.zeros(39)), dict(bias=torch.zeros(40, 1)),  # shorter than the outputs; of two dimensions
    dict(out=torch.zeros(3, 40)), dict(out=torch.zeros(2, 40, dtype=torch.bfloat16)),  # of another type; too few rows
    dict(out=torch.zeros(3, 39, dtype=torch.bfloat16)), dict(out=torch.zeros(40, 3, dtype=torch.bfloat16).t()),  # too few columns; in columns
    dict(out=torch.zeros(1, 40, dtype=torch.bfloat16).expand(3, 40)),  # every row the same
    dict(out=far(3, 40, 2 ** 31, torch.bfloat16)), dict(codes=far(40, 64, 2 ** 31, torch.int8))])  # rows too far apart
def test_what_does_not_fit_is_refused_ahead_of_the_launch(change, monkeypatch):
    """On tensors of the host, which pass for the current device's here, and without a library to launch anything."""
    from oxidize_b200.ops import cuda_int8

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1)

    def launch():
        raise AssertionError("launched")

    monkeypatch.setattr(cuda_int8, "lib", launch)
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    codes = change.get("codes", torch_quant.int8_rows(torch.zeros(40, 64, dtype=torch.int8)))
    q = QTensor("I8", codes, (40, 64), torch.ones(40))
    out = change.get("out", torch.zeros(3, 40, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        cuda_int8.linear(x, q, out, change.get("bias"), out.stride(0))
    with pytest.raises(AssertionError, match="launched"):
        cuda_int8.linear(x, QTensor("I8", torch.zeros(40, 64, dtype=torch.int8), (40, 64), torch.ones(40)), torch.zeros(4, 48, dtype=torch.bfloat16),
                         torch.zeros(41), 48)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 200])
def test_longer_biases_and_larger_outputs(T):
    """Their first values: what lies behind stays as it was."""
    gen = torch.Generator().manual_seed(41)
    q, x = weight(gen, 40, 64, "cuda"), torch.randn(T, 64, generator=gen).bfloat16().cuda()
    bias, out = torch.randn(50, generator=gen).cuda(), torch.full((T + 2, 56), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.linear(x, LinearWeight([q], bias), out=out)
    check(x, q, bias[:40], out[:T, :40])
    assert (out[T:] == 7).all() and (out[:, 40:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 300])
def test_behind_a_kernel_that_runs_for_seconds(T):
    """The product is resident while a kernel ahead of it, which let its dependents start, still runs for longer than a wait's bound of a
    second: the time of that kernel does not count."""
    from types import SimpleNamespace

    from oxidize_b200.ops import cuda as C

    gen = torch.Generator().manual_seed(43)
    q, x = weight(gen, 200, 256, "cuda"), torch.randn(T, 256, generator=gen).bfloat16().cuda()
    want = ops.linear(x, LinearWeight([q]))
    # a convolution of one channel and very many taps: one thread's work, some seconds of it
    taps = 12_000_000
    w, window, row = torch.zeros(1, taps, device="cuda"), torch.zeros(1, taps, 1, device="cuda"), torch.zeros(1, 1, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    meta = SimpleNamespace(query_start=i32(0, 1), seq_lens=i32(taps + 1), state_slots=i32(0), max_query_len=1)
    torch.cuda.synchronize()
    C.status()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    ops.causal_conv(row, w, None, meta, window, act="none")
    y = ops.linear(x, LinearWeight([q]))
    end.record()
    torch.cuda.synchronize()
    assert begin.elapsed_time(end) > 1500
    assert C.status()[0] == 0 and torch.equal(y, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1, 3, 40, 300])
def test_large_tokens(T, device):
    """Tokens around 1e35, whose sums times their scales alone would leave float32's range, with weights that bring them back."""
    gen = torch.Generator().manual_seed(44)
    x = tokens(torch.randn(T, 4096, generator=gen) * 2e35, device)
    q = qtensor_from_dense(torch.randn(200, 4096, generator=gen) * 0.02, "I8", device)
    y = ops.linear(x, LinearWeight([q]))
    assert torch.isfinite(y).all() and y.abs().max() > 1e35
    check(x, q, None, y)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 40, 300])
@pytest.mark.parametrize("k", [40959, 1023, 500, 17, 130])
def test_nothing_is_read_behind_a_row(k, T):
    """Codes between which, and behind the last of which, other codes lie in the same memory: none of them counts."""
    gen = torch.Generator().manual_seed(k)
    n, ld = 70, (k + 15) // 16 * 16
    room = torch.full((n * ld + 512,), 127, dtype=torch.int8, device="cuda")
    codes = room.as_strided((n, k), (ld, 1))
    codes.copy_(torch.randint(-127, 128, (n, k), generator=gen).to(torch.int8))
    q = QTensor("I8", codes, (n, k), (torch.rand(n, generator=gen) * 0.01).cuda())
    x = torch.randn(T, k, generator=gen).bfloat16().cuda()
    check(x, q, None, ops.linear(x, LinearWeight([q])))
