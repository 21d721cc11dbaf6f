"""Operators over sequences: the gated linear recurrence and counter-based dropout.

``gated_recurrence`` runs, per channel,

    f_t = gate_t (form="decay")  or  1 / (1 + exp(-gate_t)) (form="logit")
    h_t = f_t h_{t-1} + x_t,     coupled:  h_t = f_t h_{t-1} + (1 - f_t) x_t

over dense, padded or packed sequences, with gradients.  The rasterizer's blend is its coupled form, run from the back of a
depth-ordered list to its front with the gate 1 - alpha shared by the colour channels; here the lists may hold any number
of channels and come from anywhere:

    # samples [N, C] of all rays, front to back, ray r in rows offsets[r] .. offsets[r + 1]
    _, pixels = gated_recurrence(samples, 1 - alphas[:, None], offsets=offsets, form="decay", coupled=True, reverse=True,
                                 final_only=True)

``gated_recurrence_step`` takes one new row per sequence and updates the state in place.  ``dropout`` draws its mask from
(seed, step, element index) and never stores it; ``dp.ViewRenderer.render_views`` drops splats with it.

The reference has no counterpart of these.  Tensors are float32, float16 or bfloat16 on one CUDA device; states, sums and
all arithmetic are float32, rounded once to the tensors' type.  Work is enqueued on the current stream of the inputs'
device.  There is no fallback for other devices.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple, Union

import torch
try:
    from torch._C import _cuda_getCurrentRawStream as _raw_stream   # the current stream's handle without an object around it
except ImportError:        # a torch without CUDA: the entry points refuse its tensors before they ask for a stream
    _raw_stream = None

from . import _capi

MAX_CHANNELS = (1 << 31) - (1 << 16)   # as the library's


def _on(device, call, *args):
    """``call(*args)`` with ``device`` current (the library launches on the current device)."""
    if torch.cuda.current_device() == device.index:
        return call(*args)
    with torch.cuda.device(device):
        return call(*args)


def _require(t, name, device=None, dtype=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")


def _rows(t: torch.Tensor, lanes: int):
    """(tensor, elements between rows): ``t`` as rows of its last dimension, as it is where one stride leads from row to row
    and, for loads of ``lanes`` elements, the rows start on such boundaries; a contiguous copy otherwise."""
    width = t.shape[-1]
    if t.is_contiguous():
        plain, stride = True, width
    else:
        plain, stride, rows = t.stride(-1) == 1 or width == 1, width, 1
        for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if rows == 1:
                stride = step
            elif step != stride * rows:
                plain = False
            rows *= size
    if plain and (lanes == 1 or (stride % lanes == 0 and t.data_ptr() % (lanes * t.element_size()) == 0)):
        return t, stride
    return t.clone(memory_format=torch.contiguous_format), width


def _flat_as(t: torch.Tensor, stride: int, flat: bool):
    """``_rows``'s pair for rows that lie one behind the other exactly when ``flat``."""
    width = t.shape[-1]
    if (stride == width) == flat:
        return t, stride
    if flat:
        return t.clone(memory_format=torch.contiguous_format), width
    apart = torch.empty((t.numel() // width, width + 1), dtype=t.dtype, device=t.device)
    apart[:, :width] = t.reshape(-1, width)
    return apart, width + 1


def _state(t: Optional[torch.Tensor], shape, device, name):
    if t is None:
        return None
    if (isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.shape == shape and t.device == device and t.is_contiguous()
            and t.data_ptr() % 16 == 0):
        return t
    _require(t, name, device, torch.float32)
    if t.shape != shape:
        raise ValueError(f"{name} must have the shape {list(shape)}, got {list(t.shape)}")
    return _rows(t, 4 if shape[-1] % 4 == 0 else 2 if shape[-1] % 2 == 0 else 1)[0].contiguous()


def _check_gate(x, gate, form):
    _require(x, "x")
    if x.dtype not in _capi.DTYPES:
        raise RuntimeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    _require(gate, "gate", x.device, x.dtype)
    if form not in _capi.GATE_FORMS:
        raise ValueError(f"form must be 'decay' or 'logit', got {form!r}")
    if gate.shape != x.shape:
        if gate.dim() != x.dim() or gate.shape[:-1] != x.shape[:-1]:
            raise ValueError(f"gate must have one row per row of x: {list(gate.shape)} against {list(x.shape)}")
        d, heads = x.shape[-1], gate.shape[-1]
        if heads < 1 or d % heads != 0:
            raise ValueError(f"{d} channels do not split into {heads} gate heads")
    if not 1 <= x.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"x must have 1 to 2^31 - 2^16 channels, got {x.shape[-1]}")


_sizes = {}     # (workspace, checkpoint) bytes by what they follow from


def _lies_as_saved(t, dtype, count, index):
    """Whether ``t`` is as a contiguous tensor of these was when it was saved (and is where it was not replaced)."""
    return t.dtype is dtype and t.numel() == count and t.get_device() == index and t.is_contiguous() and t.data_ptr() % 16 == 0


class _Call:
    """What a call's forward and backward pass have in common: the DsbRecurrence (for ``x`` and ``gate`` as they are kept
    here, copied where their rows do not lie as the kernels need them) and the sizes that follow from it."""
    __slots__ = ("shape", "ref", "lanes", "x", "gate", "sequences", "final_only", "key", "sizes", "contiguous")

    def __init__(self, x, gate, sequences, sequence_rows, form, coupled, reverse, offsets, lengths, final_only=False):
        if sequences >= 1 << 31:
            raise ValueError(f"at most 2^31 - 1 sequences, got {sequences}")
        d, heads = x.shape[-1], gate.shape[-1]
        together = d // heads if heads != d else d
        self.lanes = lanes = 4 if together % 4 == 0 else 2 if together % 2 == 0 else 1
        self.x, x_stride = _rows(x, lanes)
        self.gate, gate_stride = _rows(gate, lanes if heads == d else 1)
        self.sequences, self.final_only, self.contiguous = sequences, final_only, x_stride == d and gate_stride == heads
        rows, dtype = x.numel() // d, _capi.DTYPES[x.dtype]
        self.key = (rows, sequences, sequence_rows, d, heads, dtype, x_stride, gate_stride)
        self.shape = _capi.DsbRecurrence(
            rows, sequences, sequence_rows, d, heads, dtype, _capi.GATE_FORMS[form], 1 if coupled else 0, 1 if reverse else 0, x_stride,
            gate_stride, _capi.ptr(offsets), _capi.ptr(lengths))
        self.ref = C.byref(self.shape)

    def find_sizes(self, lib):
        got = _sizes.get(self.key)
        if got is None:
            if len(_sizes) > 256:
                _sizes.clear()
            got = _sizes[self.key] = (lib.dsb_recurrence_workspace_bytes(self.ref), lib.dsb_recurrence_checkpoint_bytes(self.ref))
        self.sizes = got
        return got

    def run(self, state, keep):
        """(h or None, last, checkpoints or None)"""
        lib, x = _capi.lib(), self.x
        dev, d = x.device, x.shape[-1]
        h = None if self.final_only else torch.empty(x.shape, dtype=x.dtype, device=dev)
        last = torch.empty((self.sequences, d), dtype=torch.float32, device=dev)
        workspace_bytes, checkpoint_bytes = self.find_sizes(lib)
        checkpoints = torch.empty(checkpoint_bytes, dtype=torch.uint8, device=dev) if keep else None
        workspace = torch.empty(workspace_bytes, dtype=torch.uint8, device=dev) if workspace_bytes else None
        rc = lib.dsb_recurrence_forward(
            self.ref, x.data_ptr(), self.gate.data_ptr(), _capi.ptr(state), _capi.ptr(h), last.data_ptr(), _capi.ptr(checkpoints),
            _capi.ptr(workspace), workspace_bytes, _raw_stream(dev.index))
        if rc:
            _capi.check(rc)
        return h, last, checkpoints

    def as_handed_out(self, x, gate, state, checkpoints, borders, dev):
        """(x, gate, state, checkpoints, borders, DsbRecurrence) of a backward pass.  Hooks on saved tensors (activation
        checkpointing, offloading) hand out others than those that were saved: at other addresses, and laid out otherwise."""
        s, index, dtype = self.shape, -1 if dev.index is None else dev.index, x.dtype
        rows, sequences, sequence_rows, d, heads, code, _, _ = self.key
        packed = sequence_rows == 0
        if (self.contiguous and _capi.DTYPES.get(dtype) == code and _lies_as_saved(x, dtype, rows * d, index) and x.shape[-1] == d
                and _lies_as_saved(gate, dtype, rows * heads, index)
                and _lies_as_saved(checkpoints, torch.uint8, self.sizes[1], index)
                and (state is None or _lies_as_saved(state, torch.float32, sequences * d, index))
                and (borders is None or (_lies_as_saved(borders, torch.int32, sequences + packed, index)
                                         and borders.data_ptr() == (s.offsets if packed else s.lengths)))):
            return x, gate, state, checkpoints, borders, s      # the forward's descriptor says all of this
        for t, name, width in ((x, "x", s.channels), (gate, "gate", s.gate_heads)):
            _require(t, name, dev, x.dtype)
            if t.shape[-1] != width or t.numel() != s.rows * width or _capi.DTYPES.get(t.dtype) != s.dtype:
                raise RuntimeError(f"a hook handed out a {name} of another shape or type than was saved")
        x, x_stride = _rows(x, self.lanes)
        gate, gate_stride = _rows(gate, self.lanes if s.gate_heads == s.channels else 1)
        if s.channels == 3:     # whether rows of three are contiguous decides the cut, and with it what the checkpoints are of
            x, x_stride = _flat_as(x, x_stride, s.x_stride == 3)
            if s.gate_heads == 3:
                gate, gate_stride = _flat_as(gate, gate_stride, s.gate_stride == 3)
        state = _state(state, (self.sequences, s.channels), dev, "state")
        _require(checkpoints, "the saved states", dev, torch.uint8)
        if checkpoints.numel() != self.sizes[1]:
            raise RuntimeError("a hook handed out something else than was saved")
        if not checkpoints.is_contiguous() or checkpoints.data_ptr() % 16:
            checkpoints = checkpoints.clone(memory_format=torch.contiguous_format)
        shape = type(s).from_buffer_copy(s)
        shape.x_stride, shape.gate_stride = x_stride, gate_stride
        if borders is not None:
            _require(borders, "offsets" if packed else "lengths", dev, torch.int32)
            if borders.numel() != self.sequences + packed:
                raise RuntimeError("a hook handed out something else than was saved")
            borders = borders.contiguous()
            shape.offsets, shape.lengths = (borders.data_ptr(), None) if packed else (None, borders.data_ptr())
        return x, gate, state, checkpoints, borders, shape

    def run_backward(self, x, gate, state, checkpoints, borders, v_h, v_last, need, dev):
        lib, d = _capi.lib(), x.shape[-1]
        v_x = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
        v_gate = torch.empty(gate.shape, dtype=gate.dtype, device=dev) if need[1] else None
        x, gate, state, checkpoints, borders, shape = self.as_handed_out(x, gate, state, checkpoints, borders, dev)
        if v_h is None:
            v_h_stride = d
        elif d == 3:
            v_h, v_h_stride = v_h.contiguous(), d      # rows of three channels are copied as one piece of memory
        else:
            v_h, v_h_stride = _rows(v_h, self.lanes)
        v_last = _state(v_last, (self.sequences, d), dev, "the last state's gradient")
        v_state = torch.empty((self.sequences, d), dtype=torch.float32, device=dev) if need[2] else None
        workspace_bytes = self.sizes[0]
        workspace = torch.empty(workspace_bytes, dtype=torch.uint8, device=dev) if workspace_bytes else None
        rc = lib.dsb_recurrence_backward(
            C.byref(shape), x.data_ptr(), gate.data_ptr(), _capi.ptr(state), checkpoints.data_ptr(), _capi.ptr(v_h), v_h_stride,
            _capi.ptr(v_last), _capi.ptr(v_x), _capi.ptr(v_gate), _capi.ptr(v_state), _capi.ptr(workspace), workspace_bytes,
            _raw_stream(dev.index))
        if rc:
            _capi.check(rc)
        return v_x, v_gate, v_state


class _GatedRecurrence(torch.autograd.Function):
    """Over (x, gate, state), a ``_Call`` and the offsets or lengths its forward points at."""

    @staticmethod
    def forward(ctx, x, gate, state, call, borders):
        h, last, checkpoints = _on(x.device, call.run, state, True)
        ctx.save_for_backward(call.x, call.gate, state, checkpoints, borders)
        call.x = call.gate = None          # saved above
        ctx.call = call
        ctx.set_materialize_grads(False)
        return last if call.final_only else (h, last)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        x, gate, state, checkpoints, borders = ctx.saved_tensors
        v_h, v_last = (None, grads[0]) if len(grads) == 1 else grads
        if v_h is None and v_last is None:
            return (None,) * 5
        dev = (v_h if v_last is None else v_last).device
        v = _on(dev, ctx.call.run_backward, x, gate, state, checkpoints, borders, v_h, v_last, ctx.needs_input_grad, dev)
        return (*v, None, None)


def gated_recurrence(x: torch.Tensor, gate: torch.Tensor, state: Optional[torch.Tensor] = None, *,
                     offsets: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, form: str = "logit",
                     coupled: bool = False, reverse: bool = False,
                     final_only: bool = False) -> Tuple[Optional[torch.Tensor], torch.Tensor]:
    """Runs the recurrence over every sequence and returns ``(h, last)``: all states, in the type of ``x``, and each
    sequence's last state, float32.  Differentiable in ``x``, ``gate`` and ``state``.

    x        [B, T, D]: B sequences of T rows; with ``lengths`` (int32 [B]) only the first ``lengths[b]`` of them belong to
             sequence b.  [N, D] with ``offsets`` (int32 [S + 1], nondecreasing, within [0, N]): sequence s is rows
             ``offsets[s] .. offsets[s + 1]`` (a tile's ``ranges`` of the rasterizer are such offsets).  At most 2^31 - 2^16
             rows, as many channels, and 2^31 - 1 sequences.
    gate     x's shape with H for D: each of the H gates of a row is shared by D / H consecutive channels.  As logits
             (``form="logit"``) decays near 1 keep their precision in 16-bit types (f and 1 - f are each good to 9 * 2^-24 of
             themselves, with 16-bit logits to (9 + 1.22 |gate|) * 2^-24; a logit beyond +-87 counts as +-87); as
             ``"decay"`` they are taken as they are and are meant to lie in [-1, 1].
    state    float32 [S, D], each sequence's state before its first row; None = zeros.
    reverse  run from each sequence's last row to its first (``last`` is then the state after the first row).
    final_only  return ``(None, last)`` and do not write ``h``.

    Rows that belong to no sequence come back as zeros, their gradients too; a sequence of no rows hands its state on.
    What is not finite stays so to the end of its sequence and reaches no other sequence or channel; an infinity may become a
    NaN where the decays after it have a product below 2^-126.  Values below 2^-126 may count as zero.
    Kept for the backward pass: the inputs, and a float32 state per channel and 3 to 12 rows, all of them as saved tensors,
    so that activation checkpointing and hooks that offload them work.  No call waits for the device;
    a training step can be captured into a graph (as always with torch, while no eager graph of the same leaves lives).
    Offsets and lengths live on the device and are not read back: values out of order or range make the results invalid and
    are reported by ``dsb_take_device_status`` and by the rasterizer's calls that synchronise."""
    _check_gate(x, gate, form)
    if offsets is not None:
        if lengths is not None:
            raise ValueError("give offsets (packed rows) or lengths (padded rows), not both")
        if x.dim() != 2:
            raise ValueError(f"packed x must be [N, D], got {list(x.shape)}")
        _require(offsets, "offsets", x.device, torch.int32)
        if offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets must be one-dimensional with one entry more than there are sequences")
        offsets = offsets.contiguous()
    else:
        if x.dim() != 3:
            raise ValueError(f"x must be [B, T, D] (or [N, D] with offsets), got {list(x.shape)}")
        if lengths is not None:
            _require(lengths, "lengths", x.device, torch.int32)
            if tuple(lengths.shape) != (x.shape[0],):
                raise ValueError(f"lengths must have one entry per sequence: {list(lengths.shape)} against {x.shape[0]}")
            lengths = lengths.contiguous() if x.shape[1] else None     # no rows: nothing to cut short
    sequences = x.shape[0] if offsets is None else offsets.numel() - 1
    state = _state(state, (sequences, x.shape[-1]), x.device, "state")
    call = _Call(x, gate, sequences, x.shape[1] if offsets is None else 0, form, coupled, reverse, offsets, lengths, final_only)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (state is not None and state.requires_grad)):
        out = _GatedRecurrence.apply(call.x, call.gate, state, call, offsets if offsets is not None else lengths)
        return (None, out) if final_only else out
    return _on(x.device, call.run, state, False)[:2]


def gated_recurrence_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, *, form: str = "logit",
                          coupled: bool = False) -> torch.Tensor:
    """One row of every sequence: x [S, D], gate [S, H], ``state`` (float32 [S, D], contiguous, sharing no memory with
    them) updated in place; returns the new states in the type of ``x``.  For generating token by token; it keeps nothing
    for a backward pass."""
    _check_gate(x, gate, form)
    if x.dim() != 2:
        raise ValueError(f"x must be [S, D], got {list(x.shape)}")
    _require(state, "state", x.device, torch.float32)
    if state.shape != x.shape:
        raise ValueError(f"state must have the shape {list(x.shape)}, got {list(state.shape)}")
    if not state.is_contiguous():
        raise ValueError("state is updated in place and must be contiguous")
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or state.requires_grad):
        raise RuntimeError("gated_recurrence_step has no backward pass: use gated_recurrence, or torch.no_grad()")
    return _on(x.device, _run_step, _Call(x, gate, x.shape[0], 0, form, coupled, False, None, None), state)


def _run_step(call, state):
    x = call.x
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if h.numel():
        rc = _capi.lib().dsb_recurrence_step(call.ref, x.data_ptr(), call.gate.data_ptr(), state.data_ptr(), h.data_ptr(),
                                             _raw_stream(x.device.index))
        if rc:
            _capi.check(rc)
        torch.autograd.graph.increment_version(state)
    return h


def _launch_dropout(x, residual, p, seed, step, rng, rng_used):
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.numel() == 0:
        return out
    if x.is_contiguous() and (residual is None or residual.is_contiguous()):
        cols = x_stride = residual_stride = x.numel()
    else:
        x, x_stride = _rows(x, 1)
        cols = residual_stride = x.shape[-1]
        if residual is not None:
            residual, residual_stride = _rows(residual, 1)
    rc = _capi.lib().dsb_dropout(
        x.data_ptr(), _capi.ptr(residual), out.data_ptr(), out.numel() // cols, cols, x_stride, residual_stride, cols,
        _capi.DTYPES[x.dtype], p, seed, step, _capi.ptr(rng), _capi.ptr(rng_used), _raw_stream(x.device.index))
    if rc:
        _capi.check(rc)
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, call):
        p, seed, step, rng = call
        used = torch.empty(2, dtype=torch.int64, device=x.device) if rng is not None else None
        ctx.call = (p, seed, step, used)   # the pair as it was: the caller may advance rng before the backward pass
        return _on(x.device, _launch_dropout, x, residual, p, seed, step, rng, used)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, v_out):
        p, seed, step, used = ctx.call
        v_x = _on(v_out.device, _launch_dropout, v_out, None, p, seed, step, used, None) if ctx.needs_input_grad[0] else None
        return v_x, (v_out if ctx.needs_input_grad[1] else None), None


def dropout(x: torch.Tensor, p: float, rng: Union[Tuple[int, int], torch.Tensor], *,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[residual +] (keep ? x / (1 - p) : 0)`` with ``keep`` drawn per element with probability 1 - p from a counter-based
    generator: word i mod 4 of Philox4x32-10 with the key ``seed`` and the counter (i div 4, ``step``), i the element's
    row-major index, at least ``round(p 2^32)``.  The mask depends on nothing else and is drawn again in the backward pass.

    rng  the pair (seed, step), each within [0, 2^64): one seed per place in a model, one step per training step.  Or an
         int64 CUDA tensor of two elements holding them, read when the kernel runs: a captured graph draws a new mask at
         every replay when the tensor is advanced between (or inside) the replays.  Where activation checkpointing runs a block
         a second time, the tensor is read a second time: advance it after the backward pass, or give the pair as numbers.
    residual  a tensor of x's shape and type to add.

    Dropped elements leave no trace of what they held; p = 1 drops everything.  Values below 2^-126 may count as zero."""
    _require(x, "x")
    if x.dtype not in _capi.DTYPES:
        raise RuntimeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    if residual is not None:
        _require(residual, "residual", x.device, x.dtype)
        if residual.shape != x.shape:
            raise ValueError(f"residual must have the shape of x: {list(residual.shape)} against {list(x.shape)}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must lie in [0, 1], got {p}")
    if isinstance(rng, torch.Tensor):
        _require(rng, "rng", x.device, torch.int64)
        if rng.numel() != 2 or not rng.is_contiguous():
            raise ValueError("rng must hold two elements, (seed, step)")
        seed = step = 0
    else:
        seed, step = rng
        seed, step, rng = int(seed), int(step), None
        if not (0 <= seed < 1 << 64 and 0 <= step < 1 << 64):
            raise ValueError("seed and step must lie in [0, 2^64)")
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, (p, seed, step, rng))
    return _on(x.device, _launch_dropout, x, residual, p, seed, step, rng, None)
