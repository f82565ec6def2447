"""A residual scale without a block output is refused: the stream is only read then, and would not be scaled.  No device."""
import pytest
import torch

from mference_amd import operators as ops
from test_adapters_cpu import INVALID, LAUNCH, FakeContext, ctx, needs_no_device, norm, norm_args  # noqa: F401


@pytest.mark.parametrize("scale", [0.5, -1.0, 2.0, float("nan"), float("inf"), 1.0000001])
def test_a_scale_with_nothing_to_add_is_refused(ctx, scale, monkeypatch):  # noqa: F811
    assert norm(ctx, norm_args(delta=None, residual_scale=scale)[0]) == INVALID
    monkeypatch.setattr(ops, "_address", lambda t, *_: t.data_ptr())
    monkeypatch.setattr(ops, "_on", lambda *_: 0)
    h, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(8, dtype=torch.bfloat16)
    for value in (scale, 0.0):
        with pytest.raises(ops.MfError, match="INVALID_ARGUMENT"):
            ops.BlockNorm(FakeContext()).encode(h, out=torch.empty_like(h), pre_weight=w, residual_scale=value)


@needs_no_device
def test_the_stream_alone_is_taken(ctx):  # noqa: F811
    for scale in (1.0, 0.0):  # (0: a cleared structure)
        assert norm(ctx, norm_args(delta=None, residual_scale=scale)[0]) == LAUNCH
    for scale in (0.0, 0.5, -1.0):
        assert norm(ctx, norm_args(residual_scale=scale)[0]) == LAUNCH
