"""What the paged cache's wrappers refuse, and how they are imported, without a GPU."""
import importlib.util

import pytest
import torch

from paged_cases import normal

from moss_tts._runtime import kernels as K


def test_the_module_loads_and_finds_the_stream_without_the_private_name(monkeypatch):
    """``torch._C._cuda_getCurrentRawStream`` is not a public name: without it the public call answers."""
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    spec = importlib.util.spec_from_file_location("moss_tts._runtime.kernels_again", K.__file__)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)

    class Stream:
        cuda_stream = 1234

    asked = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: asked.append(device) or Stream())
    assert module._raw_stream(3) == 1234 and asked == [3]
