"""The Rotary module where models are built, moved and cast: its frequencies on the CPU."""
import copy

import pytest
import torch

import flare_b200 as fb

FREQS = 10_000.0 ** -(torch.arange(0, 16, 2, dtype=torch.float64) / 16)


def right(rope, device="cpu"):
    assert rope.freqs.dtype == torch.float64 and rope.freqs.device.type == device and not rope.state_dict()
    assert device == "meta" or torch.equal(rope.freqs, FREQS)


def test_built_without_memory_and_materialised():
    with torch.device("meta"):
        net = torch.nn.Sequential(torch.nn.Linear(16, 16), fb.Rotary(16))
        f, _ = fb.rotary_frequencies(16)
    assert f.device.type == "cpu" and torch.equal(f, FREQS)
    right(net[1], "meta")
    net.to_empty(device="cpu")
    right(net[1])
    right(copy.deepcopy(net)[1])
    right(fb.Rotary(16).to("meta"), "meta")
    right(fb.Rotary(16).to("meta").to_empty(device="cpu"))


def test_the_default_device_is_the_buffers_not_the_functions():
    with torch.device("meta"):
        assert fb.Rotary(16).freqs.device.type == "meta"
    torch.set_default_device("meta")
    try:
        assert fb.rotary_frequencies(16, scaling="by_parts", factor=2.0, original_length=64)[0].device.type == "cpu"
    finally:
        torch.set_default_device(None)


def test_a_move_that_is_none_leaves_the_buffer_where_it_is():
    """A captured graph reads the frequencies at their address: casting a model, or moving it to where it is, must not change it."""
    rope = fb.Rotary(16)
    at = rope.freqs.data_ptr()
    net = torch.nn.Sequential(rope)
    for move in (lambda: net.half(), lambda: net.float(), lambda: net.to("cpu"), lambda: net.to(torch.bfloat16), lambda: net.double(),
                 lambda: net.cpu(), lambda: net.to_empty(device="cpu")):
        move()
        right(rope)
        assert rope.freqs.data_ptr() == at
    net.share_memory()
    assert rope.freqs.is_shared()
    right(rope)
    # and what a user does to the buffer of one module stays with it
    other = fb.Rotary(16).to("meta").to_empty(device="cpu")
    other.freqs.zero_()
    right(other.to("meta").to_empty(device="cpu"))


@pytest.mark.gpu
def test_a_captured_graph_outlives_a_move_to_the_same_device(cuda_dev):
    rope = fb.Rotary(16).to(cuda_dev)
    x = torch.randn(1, 2, 9, 16, device=cuda_dev)
    rope(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rope(x)
    at = rope.freqs.data_ptr()
    rope.to(cuda_dev).half().float()
    assert rope.freqs.data_ptr() == at
    fill = [torch.full((8,), 7.0, dtype=torch.float64, device=cuda_dev) for _ in range(64)]   # whatever was freed is used again
    graph.replay()
    assert torch.equal(y, rope(x)) and len(fill) == 64
