"""The current stream's handle, with and without torch's short way to it."""
import importlib.util
import sys

import pytest
import torch

import fmkv


def test_without_the_short_way(monkeypatch):
    """A torch without the name still gives the stream (no GPU needed)."""
    class Current:
        cuda_stream = 77

    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Current())
    spec = importlib.util.spec_from_file_location("fmkv_again", fmkv.__file__)
    again = importlib.util.module_from_spec(spec)
    monkeypatch.setitem(sys.modules, "fmkv_again", again)
    spec.loader.exec_module(again)
    assert again._stream(None) == 77 and again._stream(5) == 5 and again._stream(Current()) == 77


@pytest.mark.gpu
def test_both_ways_agree(gpu, monkeypatch):
    side = torch.cuda.Stream()
    for short in (gpu._raw_stream, None):
        monkeypatch.setattr(gpu, "_raw_stream", short)
        assert gpu._stream(None) == torch.cuda.current_stream().cuda_stream
        with torch.cuda.stream(side):
            assert gpu._stream(None) == side.cuda_stream != torch.cuda.default_stream().cuda_stream
        assert gpu._stream(side) == side.cuda_stream
