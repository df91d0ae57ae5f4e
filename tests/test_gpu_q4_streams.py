"""A 4-bit head made on one stream and used, and dropped, on others."""
import pytest
import torch

from tests.test_gpu_q4 import parts, states

pytestmark = pytest.mark.gpu


def _ctx():
    from tests.gpu_util import ctx
    return ctx()


def _busy(n=20):
    """Some milliseconds of work on the current stream."""
    x = torch.ones((4096, 4096), device="cuda")
    for _ in range(n):
        x = x @ x * 2.0 ** -12
    return x


def test_used_on_another_stream_at_once():
    """Made behind work of its own stream; another stream's first call finds it whole."""
    from zllm_amd.head import Q4Head
    p = parts(100000, 512, 64, True)
    hs = [states(3, 512, "bf16"), states(40, 512, "f32")]
    want = [Q4Head(_ctx(), *p).logits(h) for h in hs]
    torch.cuda.synchronize()
    made, used = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(made):
            _busy()
            head = Q4Head(_ctx(), *p)
        with torch.cuda.stream(used):
            got = [head.logits(h) for h in hs]
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_dropped_while_another_stream_is_to_read_it():
    """The stream that made it gets its memory back when the other is through."""
    from zllm_amd.head import Q4Head
    p = parts(100000, 512, 64, True)
    h = states(3, 512, "bf16")
    head = Q4Head(_ctx(), *p)
    want = head.logits(h)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        head = Q4Head(_ctx(), *p)
        nbytes, at = head._data.numel(), head._data.data_ptr()
        with torch.cuda.stream(side):
            _busy()
            got = head.logits(h)
        del head
        other = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
        assert other.data_ptr() != at
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del other


def test_many_calls_on_streams_keep_one_note_of_each():
    from zllm_amd.head import Q4Head
    head = Q4Head(_ctx(), *parts(1000, 128, 32, False))
    h = states(3, 128, "bf16")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams * 4:
        with torch.cuda.stream(s):
            head.logits(h)
    torch.cuda.synchronize()
    assert head._streams == {torch.cuda.current_stream().cuda_stream, *(s.cuda_stream for s in streams)}


def test_made_in_a_captured_graph():
    """Quantised, laid out and used in a graph: replayed, it follows the weight."""
    from zllm_amd.head import Q4Head
    gen = torch.Generator("cuda").manual_seed(1)
    W = torch.randn((3000, 256), device="cuda", generator=gen)
    h = states(5, 256, "bf16")
    Q4Head.quantize(_ctx(), W, 64).logits(h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        head = Q4Head.quantize(_ctx(), W, 64)
        out = head.logits(h)
    for seed in range(4):
        W.copy_(torch.randn((3000, 256), device="cuda", generator=gen))
        h.copy_(states(5, 256, "bf16", seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        want = Q4Head.quantize(_ctx(), W, 64).logits(h)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_used_in_a_captured_graph_that_another_stream_replays():
    from zllm_amd.head import Q4Head
    head = Q4Head(_ctx(), *parts(3000, 256, 32, False))
    h = states(40, 256, "f32")
    head.logits(h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = head.logits(h)
    side = torch.cuda.Stream()
    for seed in range(4):
        h.copy_(states(40, 256, "f32", seed=seed))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, head.logits(h))
