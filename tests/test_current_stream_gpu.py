"""The stream that launches from Python go to."""
import pytest
import torch

from vosti_amd.kernels import kernels_for, ops

pytestmark = pytest.mark.gpu


def test_the_current_stream_by_either_name(monkeypatch):
    """Where torch has no private name for it a launch goes to the same stream."""
    k = kernels_for("bf16")
    for st in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(st):
            with monkeypatch.context() as m:
                m.setattr(ops, "_raw_stream", None)
                assert k._stream() == st.cuda_stream
            assert k._stream() == st.cuda_stream
