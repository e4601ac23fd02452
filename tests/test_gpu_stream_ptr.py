"""Stream handles of the binding: torch's own, whatever stream is current."""
import pytest

import dramamoe as D

pytestmark = pytest.mark.gpu


def test_current_stream():
    import torch

    assert D.stream_ptr() == torch.cuda.current_stream().cuda_stream
    for st in (torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.default_stream()):
        assert D.stream_ptr(st) == st.cuda_stream
        with torch.cuda.stream(st):
            assert D.stream_ptr() == st.cuda_stream == torch.cuda.current_stream().cuda_stream
    assert D.stream_ptr() == torch.cuda.current_stream().cuda_stream
