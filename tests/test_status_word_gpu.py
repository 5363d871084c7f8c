"""The single-GPU operators' device status word: ready for every stream, and a launch that found it set says so."""
import pytest
import torch

import paraattention_b200 as pa
from paraattention_b200 import _lib as L
from paraattention_b200 import _status, ops

pytestmark = pytest.mark.gpu


def make(B=2, H=2, Sq=200, Skv=150, D=64, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(B, s, H, D, device="cuda", generator=g).bfloat16().transpose(1, 2) for s in (Sq, Skv, Skv)]


@pytest.mark.parametrize("backward", [False, True])
def test_a_launch_that_returned_at_its_entry_is_raised_by_the_next_call(backward):
    """The device's word alone is set, as by a wait that gave up under another status mirror's eyes: the launch that finds it
    leaves its outputs alone, and says so in the host's word."""
    q, k, v = (t.requires_grad_(True) for t in make())
    out = ops.cross_attention(q, k, v)
    want = torch.autograd.grad(out, (q, k, v), torch.ones_like(out), retain_graph=True)
    mirror = _status.single_gpu_status(q.device)
    torch.cuda.synchronize()
    try:
        mirror.word.fill_(L.PA_DEV_TIMEOUT_PIPE)
        if backward:
            torch.autograd.grad(out, (q, k, v), torch.ones_like(out), retain_graph=True)
        else:
            ops.cross_attention(q.detach(), k.detach(), v.detach())
        torch.cuda.synchronize()
        with pytest.raises(L.PaError) as e:
            ops.cross_attention(q.detach(), k.detach(), v.detach())
        assert e.value.code == L.PA_ETIMEDOUT
        with pytest.raises(L.PaError):
            pa.check_device_status()
    finally:
        torch.cuda.synchronize()
        pa.reset_device_status()
    pa.check_device_status()
    again = torch.autograd.grad(ops.cross_attention(q, k, v), (q, k, v), torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_the_status_word_is_ready_for_every_stream():
    """Made on a stream that is busy, where memory is at hand that held something else: another stream reads it at once."""
    dev = torch.device("cuda", torch.cuda.current_device())
    kept = dict(_status._single)
    side = torch.cuda.Stream()
    try:
        _status._single.clear()
        with torch.cuda.stream(side):
            junk = torch.full((1,), 7, dtype=torch.int32, device=dev)
            side.synchronize()
            del junk
            torch.cuda._sleep(400_000_000)
            mirror = _status.single_gpu_status(dev)
        seen = int(mirror.word.item())  # on this stream
        assert seen == 0
        side.synchronize()
    finally:
        _status._single.clear()
        _status._single.update(kept)


def test_a_first_call_inside_a_capture_keeps_its_word_to_itself():
    """ops.attention_forward makes a word where it is called. Inside a capture the fill is the graph's, so launches outside,
    which may run before any replay, have another."""
    q, k, v = make(Sq=300)
    want, cross = ops.attention_forward(q, q, q), ops.cross_attention(q, k, v)
    torch.cuda.synchronize()
    kept, graphs = dict(_status._single), list(_status._in_graphs)
    try:
        _status._single.clear()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.attention_forward(q, q, q)
        assert not _status._single and len(_status._in_graphs) == len(graphs) + 1
        assert _status._in_graphs[-1] in _status.all_mirrors()
        assert torch.equal(ops.cross_attention(q, k, v), cross) and torch.equal(ops.attention_forward(q, q, q), want)
        assert _status._single[q.device.index].word.data_ptr() != _status._in_graphs[-1].word.data_ptr()
        for _ in range(2):
            graph.replay()
        assert torch.equal(out, want)
        pa.check_device_status()
    finally:
        torch.cuda.synchronize()
        _status._single.clear()
        _status._single.update(kept)


def test_a_first_call_in_inference_mode():
    """The status words it makes serve calls and resets outside of inference mode, too."""
    dev = torch.device("cuda", torch.cuda.current_device())
    kept = dict(_status._single)
    q, k, v = make()
    want = ops.cross_attention(q, k, v)
    try:
        _status._single.clear()
        with torch.inference_mode():
            assert torch.equal(ops.cross_attention(q, k, v), want)
        ops.attention_forward(q, q, q)  # (queues a copy to the host's word)
        assert torch.equal(ops.cross_attention(q, k, v), want)
        torch.cuda.synchronize()
        pa.reset_device_status()
        assert torch.equal(ops.cross_attention(q, k, v), want) and dev.index in _status._single
    finally:
        torch.cuda.synchronize()
        _status._single.clear()
        _status._single.update(kept)
