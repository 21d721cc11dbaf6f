"""Sizes that the recurrence's entry points refuse, on the CPU: no channels, and counts beyond what its descriptor holds."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import ds_splat_b200 as ds  # noqa: E402
from ds_splat_b200 import _capi, sequence  # noqa: E402
from test_sequence_host import lib, shape_of  # noqa: E402, F401


@pytest.fixture
def no_device_check(monkeypatch):
    def refuse():
        raise AssertionError("the library must not be called")

    monkeypatch.setattr(sequence, "_require", lambda *a, **k: None)
    monkeypatch.setattr(_capi, "lib", refuse)


@pytest.mark.parametrize("heads", [0, 1, 2])
def test_no_channels(no_device_check, heads):
    with pytest.raises(ValueError, match="channel|heads"):
        ds.gated_recurrence(torch.zeros(2, 3, 0), torch.zeros(2, 3, heads))
    with pytest.raises(ValueError, match="channel|heads"):
        ds.gated_recurrence_step(torch.zeros(2, 0), torch.zeros(2, heads), torch.zeros(2, 0))


@pytest.mark.parametrize("count", [1 << 31, (1 << 32) + 2])
def test_more_sequences_than_the_descriptor_counts(no_device_check, count):
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="sequences"):
        sequence._Call(x, x, count, 0, "logit", False, False, torch.zeros(1, dtype=torch.int32), None)


@pytest.mark.parametrize("count", [(1 << 31) - (1 << 16) + 1, 1 << 31, (1 << 32) + 8])
def test_more_channels_than_the_descriptor_counts(no_device_check, count):
    x = torch.zeros(1).expand(2, 1, count)           # one element, read again and again
    with pytest.raises(ValueError, match="channels"):
        ds.gated_recurrence(x, x)


def test_the_c_entry_points_refuse_channels_beyond_their_arithmetic(lib):  # noqa: F811
    shape = shape_of(rows=1, sequences=1, sequence_rows=1, channels=(1 << 31) - 8, heads=(1 << 31) - 8, x_stride=0, gate_stride=0)
    assert lib.dsb_recurrence_forward(C.byref(shape), 256, 256, None, 256, 512, None, 256, 1 << 20, None) == -1
    assert "channels" in lib.dsb_last_error().decode()
    assert lib.dsb_recurrence_checkpoint_bytes(C.byref(shape)) == 0
