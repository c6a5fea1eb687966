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
