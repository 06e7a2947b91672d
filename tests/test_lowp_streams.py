"""Outputs that quantize_i8 and newton_schulz make themselves, when the call runs on another stream than the current one: they
are the writing stream's memory (a block of the current stream's pool may still be read by what is queued there), and the
allocator is told that the current stream uses them too."""
import contextlib

import pytest

torch = pytest.importorskip("torch")

from batchlas_b200 import orthogonal, quantized  # noqa: E402

CURRENT, SIDE = 0, 77


class Stream:
    def __init__(self, raw, device=None):
        self.cuda_stream = raw


class Array:
    """What the Python layer asks of a CUDA tensor."""
    device = torch.device("cuda", 0)

    def __init__(self, shape, dtype, made_on):
        self.shape, self.dtype, self.made_on, self.used_on = torch.Size(shape), dtype, made_on, []

    def get_device(self):
        return 0

    def stride(self):
        return torch.empty(self.shape, device="meta").stride()

    def data_ptr(self):
        return 1 << 20

    def numel(self):
        return self.shape.numel()

    def record_stream(self, stream):
        self.used_on.append(stream.cuda_stream)


@pytest.fixture
def made(monkeypatch, lib):
    """The arrays that torch.empty makes, by a fake of torch's streams and allocator; no launch."""
    stack, arrays = [Stream(CURRENT)], []
    real = torch.empty

    def empty(*shape, dtype=None, device=None, **kw):
        if device == "meta":
            return real(*shape, dtype=dtype, device=device)
        arrays.append(Array(shape[0] if not isinstance(shape[0], int) else shape, dtype, stack[-1].cuda_stream))
        return arrays[-1]

    @contextlib.contextmanager
    def on(stream):
        stack.append(stream)
        yield
        stack.pop()

    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: Stream(0))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: stack[-1])
    for module in (quantized, orthogonal):
        monkeypatch.setattr(module, "_launch", lambda *a: None)
    return arrays


@pytest.mark.parametrize("stream", [None, CURRENT, SIDE])
def test_outputs_belong_to_the_stream_that_writes_them(made, stream):
    x = Array((3, 40, 64), torch.float32, CURRENT)
    q, scale = quantized.quantize_i8(x, stream=stream)
    y = orthogonal.newton_schulz(x, stream=stream)
    writer = CURRENT if stream is None else stream
    assert q in made and scale in made and y in made
    assert all(a.made_on == writer for a in made)
    for out in (q, scale, y):
        assert out.used_on == ([CURRENT] if writer != CURRENT else [])


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["quantize", "orthogonalise"])
def test_a_block_that_queued_work_still_reads_is_not_written(lib, call):
    import batchlas_b200 as bl
    x = torch.randn(64, 4096, generator=torch.Generator().manual_seed(1)).cuda()
    side = torch.cuda.Stream()
    sizes = [64 * 4096, 64 * 4] if call == "quantize" else [64 * 4096 * 4]     # bytes of Q and scale, of Y
    want = bl.quantize_i8(x) if call == "quantize" else (bl.newton_schulz(x),)
    torch.cuda.synchronize()
    old = [torch.full((n,), 0x5a, dtype=torch.uint8, device="cuda") for n in sizes]
    copies = [torch.empty_like(o) for o in old]
    torch.cuda.synchronize()
    torch.cuda._sleep(40_000_000)                       # about 20 ms before the copies start
    for c, o in zip(copies, old):
        c.copy_(o)
    del old, o
    got = bl.quantize_i8(x, stream=side.cuda_stream) if call == "quantize" else (bl.newton_schulz(x, stream=side.cuda_stream),)
    torch.cuda.synchronize()
    assert all(bool((c == 0x5a).all()) for c in copies)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    assert bl.device_status() == 0


@pytest.mark.gpu
def test_outputs_made_on_a_side_stream_of_a_capture(lib):
    import batchlas_b200 as bl
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(40, 512, generator=gen).cuda()
    side = torch.cuda.Stream()
    bl.quantize_i8(x), bl.newton_schulz(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        q, s = bl.quantize_i8(x, stream=side.cuda_stream)
        y = bl.newton_schulz(x, stream=side.cuda_stream)
        for _ in range(3):                       # dropped at once
            bl.quantize_i8(x, stream=side.cuda_stream), bl.newton_schulz(x, stream=side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        values = q * s[:, None]
    for _ in range(3):
        x.copy_(torch.randn(40, 512, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        want_q, want_s = bl.quantize_i8(x)
        assert torch.equal(q, want_q) and torch.equal(s, want_s) and torch.equal(values, want_q * want_s[:, None])
        assert torch.equal(y, bl.newton_schulz(x))
    assert bl.device_status() == 0
