"""The sequence operators without a GPU: the checker against published words and against differences, the refusals of the
Python entry points and of the C entry points (argument checks that fail before any CUDA call), the sizes they report."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ds_splat_b200 as ds  # noqa: E402
from ds_splat_b200 import _capi  # noqa: E402
from ds_splat_b200.dp import SplatDropout  # noqa: E402
from ds_splat_b200.sequence import _rows  # noqa: E402
from oracle import sequence_oracle as O  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    import os
    from ds_splat_b200 import build
    if not os.path.exists(_capi.LIB_PATH):
        build.build()
    return _capi.lib()


def test_generator_of_the_checker_gives_the_published_words():
    # the known-answer words that were published with the generator
    assert [int(w) for w in O.philox_words(4, 0, 0)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    full = (1 << 64) - 1
    block = O.philox_words(4, full, full, first=0)     # key and high counter words of all ones, low counter 0
    assert len(set(int(w) for w in block)) == 4
    # a stretch that begins later is a stretch of the whole
    assert np.array_equal(O.philox_words(24, 7, 9)[8:], O.philox_words(16, 7, 9, first=8))


@pytest.mark.parametrize("form", ["logit", "decay"])
@pytest.mark.parametrize("coupled", [False, True])
@pytest.mark.parametrize("reverse", [False, True])
def test_gradients_of_the_checker_agree_with_differences(form, coupled, reverse):
    r = np.random.RandomState(3)
    begin, count, n, d, heads = [1, 4, 4, 9], [3, 0, 5, 1], 11, 6, 2
    x, state = r.randn(n, d), r.randn(4, d)
    gate = r.randn(n, heads) if form == "logit" else r.uniform(-1, 1, (n, heads))
    v_h, v_last = r.randn(n, d), r.randn(4, d)
    inside = np.zeros((n, 1))
    for b, c in zip(begin, count):
        inside[b:b + c] = 1

    def loss(x, gate, state):
        o = O.recurrence(x, gate, state, begin, count, form, coupled, reverse)
        return (o["h"][0] * v_h * inside).sum() + (o["last"][0] * v_last).sum()

    got = O.recurrence(x, gate, state, begin, count, form, coupled, reverse, v_h, v_last)
    for name, at in (("dx", 0), ("dgate", 1), ("dstate", 2)):
        args = [x, gate, state]
        grad = got[name][0]
        for index in np.ndindex(*args[at].shape):
            step, values = 1e-6, []
            for sign in (1, -1):
                moved = args[at].copy()
                moved[index] += sign * step
                values.append(loss(*[moved if k == at else a for k, a in enumerate(args)]))
            slope = (values[0] - values[1]) / (2 * step)
            # the third derivative's share is below step^2 times a few units; rounding is 2^-53 of the loss over the step
            assert abs(slope - grad[index]) < 1e-7 * (1 + abs(slope)), (name, index)


def test_python_entry_points_refuse_cpu_tensors_and_bad_arguments():
    x, g = torch.zeros(2, 3, 4), torch.zeros(2, 3, 4)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ds.gated_recurrence(x, g)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ds.gated_recurrence_step(x[0], g[0], x[0])
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ds.dropout(x, 0.1, (0, 0))
    with pytest.raises(TypeError):
        ds.gated_recurrence(None, g)
    with pytest.raises(TypeError):
        ds.dropout([1.0], 0.1, (0, 0))
    for bad in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            SplatDropout(bad, 0)
    with pytest.raises(ValueError):
        SplatDropout(0.5, -1)
    with pytest.raises(ValueError):
        SplatDropout(0.5, 0, 1 << 64)


def test_rows_are_taken_as_they_lie_where_one_stride_leads_through_them():
    wide = torch.arange(2 * 3 * 16.0).view(2, 3, 16)
    t, stride = _rows(wide[..., 4:8], 4)
    assert t.data_ptr() == wide[..., 4:8].data_ptr() and stride == 16
    t, stride = _rows(wide[..., 1:5], 4)                       # not on a boundary of four: copied
    assert stride == 4 and torch.equal(t, wide[..., 1:5]) and t.is_contiguous()
    t, stride = _rows(wide[..., 1:5], 1)
    assert t.data_ptr() == wide[..., 1:5].data_ptr() and stride == 16
    t, stride = _rows(wide[:, :2], 1)                          # rows of the two sequences do not follow one stride
    assert stride == 16 and t.is_contiguous() and torch.equal(t, wide[:, :2])
    t, stride = _rows(wide[:1, :2], 1)
    assert t.data_ptr() == wide.data_ptr() and stride == 16
    t, stride = _rows(wide.transpose(1, 2), 1)
    assert stride == 3 and t.is_contiguous() and torch.equal(t, wide.transpose(1, 2))
    t, stride = _rows(torch.zeros(4).expand(5, 4), 4)          # one row read again and again
    assert stride == 0 and tuple(t.shape) == (5, 4)
    t, stride = _rows(torch.zeros(7, 3)[:, 1:2], 1)            # one column: its own stride says nothing
    assert stride == 3
    t, stride = _rows(torch.zeros(3).expand(1, 1, 3)[:, :, :1], 1)
    assert stride == 1


def shape_of(rows=12, sequences=3, sequence_rows=4, channels=8, heads=8, dtype=0, form=1, x_stride=8, gate_stride=8, offsets=None,
             lengths=None):
    return _capi.DsbRecurrence(rows, sequences, sequence_rows, channels, heads, dtype, form, 0, 0, x_stride, gate_stride, offsets, lengths)


@pytest.mark.parametrize("change, text", [
    (dict(dtype=7), "dtype"), (dict(form=2), "form"), (dict(channels=0), "channels"), (dict(heads=3), "heads"),
    (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(rows=13), "rows"), (dict(sequences=-1), "sequences"),
    (dict(sequence_rows=0), "offsets"), (dict(sequence_rows=-4), "sequence_rows"), (dict(offsets=64), "offsets"),
    (dict(sequence_rows=0, offsets=64, lengths=64), "lengths"), (dict(x_stride=9), "boundary"), (dict(gate_stride=6), "boundary"),
])
def test_c_entry_points_refuse_bad_shapes(lib, change, text):
    """Every pointer here is a made-up address that the calls must not get as far as using."""
    shape = shape_of(**change)
    for call in (lambda: lib.dsb_recurrence_forward(C.byref(shape), 256, 256, None, 256, 512, None, 256, 1 << 20, None),
                 lambda: lib.dsb_recurrence_backward(C.byref(shape), 256, 256, None, 256, 256, 8, None, 256, 256, None, 256, 1 << 20, None)):
        assert call() == -1
        assert text in lib.dsb_last_error().decode()
    if not {"boundary"} & {text}:
        assert lib.dsb_recurrence_workspace_bytes(C.byref(shape)) == 0
        assert lib.dsb_recurrence_checkpoint_bytes(C.byref(shape)) == 0


def test_c_entry_points_refuse_null_pointers_small_workspaces_and_misaligned_tensors(lib):
    shape = shape_of(rows=4000, sequences=1, sequence_rows=4000)
    need = lib.dsb_recurrence_workspace_bytes(C.byref(shape))
    assert need > 0 and lib.dsb_recurrence_checkpoint_bytes(C.byref(shape)) > 0
    forward = lambda **k: lib.dsb_recurrence_forward(  # noqa: E731
        C.byref(shape), k.get("x", 256), k.get("gate", 256), k.get("state", None), k.get("h", 256), k.get("last", 512), None,
        k.get("ws", 256), k.get("bytes", need), None)
    assert lib.dsb_recurrence_forward(None, 256, 256, None, 256, 512, None, 256, need, None) == -1
    for k in (dict(x=None), dict(gate=None), dict(last=None), dict(state=512), dict(x=260), dict(gate=264), dict(h=258),
              dict(state=1028), dict(last=1028), dict(ws=264)):
        assert forward(**k) == -1, k
    assert forward(bytes=16) == -3 and forward(ws=None) == -3
    assert "workspace" in lib.dsb_last_error().decode()
    backward = lambda **k: lib.dsb_recurrence_backward(  # noqa: E731
        C.byref(shape), 256, 256, None, k.get("marks", 256), 256, k.get("stride", 8), k.get("v_last", None), k.get("v_x", 256),
        k.get("v_gate", 256), k.get("v_state", None), 256, k.get("bytes", need), None)
    colours = shape_of(rows=4, sequences=1, sequence_rows=4, channels=3, heads=1, x_stride=3, gate_stride=1)
    assert lib.dsb_recurrence_backward(C.byref(colours), 256, 256, None, 256, 256, 5, None, 256, 256, None, 256, 1 << 20, None) == -1
    assert "contiguous" in lib.dsb_last_error().decode()
    for k in (dict(marks=None), dict(marks=264), dict(stride=9), dict(v_last=512, v_state=512), dict(v_x=260), dict(v_gate=260)):
        assert backward(**k) == -1, k
    assert backward(bytes=0) == -3
    step = shape_of(rows=3, sequences=2, sequence_rows=0)
    assert lib.dsb_recurrence_step(C.byref(step), 256, 256, 512, 256, None) == -1
    step = shape_of(rows=2, sequences=2, sequence_rows=0)
    for args in ((None, 256, 512, 256), (256, None, 512, 256), (256, 256, None, 256), (256, 256, 512, None), (260, 256, 512, 256),
                 (256, 256, 516, 256)):
        assert lib.dsb_recurrence_step(C.byref(step), *args, None) == -1
    assert lib.dsb_recurrence_step(None, 256, 256, 512, 256, None) == -1
    # one shared gate is read value by value and may lie anywhere
    shape = shape_of(rows=2, sequences=2, sequence_rows=0, heads=1, gate_stride=3)
    assert lib.dsb_recurrence_step(C.byref(shape), 260, 258, 512, 256, None) == -1 and "x must" in lib.dsb_last_error().decode()


def test_c_dropout_refuses_bad_arguments(lib):
    call = lambda x=256, out=256, rows=2, cols=8, dtype=0, p=0.5: lib.dsb_dropout(  # noqa: E731
        x, None, out, rows, cols, cols, cols, cols, dtype, p, 0, 0, None, None, None)
    for k in (dict(x=None), dict(out=None), dict(rows=-1), dict(cols=-1), dict(dtype=3), dict(p=-0.1), dict(p=1.1),
              dict(p=float("nan")), dict(rows=1 << 40, cols=1 << 40)):
        assert call(**k) == -1, k
    assert call(rows=0, x=None, out=None) == 0      # nothing to do


def test_nothing_to_scan_is_not_an_error(lib):
    assert lib.dsb_recurrence_forward(C.byref(shape_of(rows=0, sequences=0)), None, None, None, None, None, None, None, 0, None) == 0
    assert lib.dsb_recurrence_step(C.byref(shape_of(rows=0, sequences=0)), None, None, None, None, None) == 0
