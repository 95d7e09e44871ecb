"""How calls find the stream that they go to."""

from __future__ import annotations

import pytest
import torch

from mini_inference_engine_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", [None, 0, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0)], ids=str)
def test_a_device_by_any_name(name):
    """A device, its ordinal or its name, as ``torch.cuda.current_stream`` takes them."""

    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            assert (_lib.stream_arg(name).value or 0) == stream.cuda_stream
