"""The recurrence's backward pass where hooks on saved tensors (activation checkpointing, offloading) hand it other tensors than
the forward pass saved: at other addresses and laid out otherwise.  On the CPU a stand-in for the library shows what it is
given; on the GPU the gradients have to be those of a plain call, bit for bit."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import ds_splat_b200 as ds  # noqa: E402
from ds_splat_b200 import _capi, sequence  # noqa: E402
from torch.utils.checkpoint import checkpoint  # noqa: E402


def anew(t):
    """The same values in other memory, contiguous: what offloading to the host and back gives."""
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def spread_out(t):
    """The same values in other memory, rows further apart and beginning off every boundary."""
    if t.dim() < 2:
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].copy_(t)
    room = torch.empty((*t.shape[:-1], t.shape[-1] + 3), dtype=t.dtype, device=t.device)
    return room[..., 1:t.shape[-1] + 1].copy_(t)


def row_stride(t):
    """Elements from row to row, None where no single stride leads through the rows."""
    if t.is_contiguous():
        return t.shape[-1]
    return sequence._rows(t, 1)[1] if sequence._rows(t, 1)[0] is t else None


class Library:
    """Stands in for the library on the CPU: keeps what its calls were given and computes nothing."""

    def __init__(self):
        self.backward = []

    def dsb_recurrence_workspace_bytes(self, ref):
        return 64

    def dsb_recurrence_checkpoint_bytes(self, ref):
        return 256

    def dsb_recurrence_forward(self, *args):
        return 0

    def dsb_recurrence_backward(self, ref, x, gate, state, checkpoints, v_h, v_h_stride, v_last, *results):
        s = ref._obj
        self.backward.append(dict(x=x, gate=gate, state=state, checkpoints=checkpoints, offsets=s.offsets, lengths=s.lengths,
                                  x_stride=s.x_stride, gate_stride=s.gate_stride, reverse=s.reverse, rows=s.rows))
        return 0


@pytest.fixture
def library(monkeypatch):
    stand_in = Library()

    def require(t, name, device=None, dtype=None):
        if (device is not None and t.device != device) or (dtype is not None and t.dtype != dtype):
            raise RuntimeError(f"{name}: {t.device}, {t.dtype}")

    monkeypatch.setattr(_capi, "lib", lambda: stand_in)
    monkeypatch.setattr(sequence, "_on", lambda device, call, *args: call(*args))
    monkeypatch.setattr(sequence, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(sequence, "_require", require)
    monkeypatch.setattr(sequence, "_sizes", {})
    return stand_in


def run_with_hooks(unpack, d, heads, dtype, layout, sliced, library):
    """What the library was given in the backward pass, and the tensors that the hooks handed out, all still alive."""
    wide = torch.randn(2, 50, 2 * d, dtype=torch.float32).to(dtype)
    gates = torch.randn(2, 50, 2 * heads, dtype=torch.float32).to(dtype)
    x, gate = (wide[..., d:], gates[..., heads:]) if sliced else (wide[..., d:].contiguous(), gates[..., heads:].contiguous())
    more = {}
    if layout == "packed":
        x, gate = x.flatten(0, 1), gate.flatten(0, 1)
        more["offsets"] = torch.tensor([0, 40, 100], dtype=torch.int32)
    elif layout == "padded":
        more["lengths"] = torch.tensor([50, 7], dtype=torch.int32)
    x, gate, state = x.requires_grad_(), gate.requires_grad_(), torch.randn(2, d).requires_grad_()
    handed = []

    def hand_out(t):
        handed.append(unpack(t))
        return handed[-1]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.preserve_format), hand_out):
        h, last = ds.gated_recurrence(x, gate, state, **more)
    torch.autograd.grad([h, last], [x, gate, state], [torch.zeros_like(h), torch.zeros_like(last)])
    return library.backward.pop(), handed, row_stride(x), row_stride(gate)


@pytest.mark.parametrize("unpack", [anew, spread_out])
@pytest.mark.parametrize("layout", ["dense", "padded", "packed"])
@pytest.mark.parametrize("sliced", [False, True])
@pytest.mark.parametrize("d, heads, dtype", [(8, 8, torch.float32), (12, 3, torch.bfloat16), (5, 5, torch.float16), (3, 3, torch.float32),
                                             (3, 1, torch.float32)])
def test_the_backward_pass_takes_the_tensors_that_hooks_hand_out(library, unpack, layout, sliced, d, heads, dtype):
    got, handed, x_stride, gate_stride = run_with_hooks(unpack, d, heads, dtype, layout, sliced, library)
    x, gate, state, checkpoints = handed[:4]
    lanes = 1 if d == 3 else 4 if (d // heads if heads != d else d) % 4 == 0 else 1
    # x and the gate: as they were handed out where their rows lie as the kernels need them, with their own stride; a copy otherwise,
    # which the stand-in cannot look into, but whose stride says how it may be read
    for name, t, need in (("x", x, lanes), ("gate", gate, lanes if heads == d else 1)):
        fits = row_stride(t) is not None and (need == 1 or (row_stride(t) % need == 0 and t.data_ptr() % (need * t.element_size()) == 0))
        if got[name] == t.data_ptr():
            assert fits and got[name + "_stride"] == row_stride(t)
        else:
            assert not fits or d == 3, "copied without need"
            assert got[name + "_stride"] in (t.shape[-1], t.shape[-1] + 1)
    # contiguous rows of three are cut otherwise than others: the checkpoints are those of the forward's cut
    if d == 3:
        flat = x_stride == 3 and (heads == 1 or gate_stride == 3)
        assert (got["x_stride"] == 3 and (heads == 1 or got["gate_stride"] == 3)) == flat
    if layout != "dense":
        borders = handed[-1]
        assert got["offsets" if layout == "packed" else "lengths"] == borders.data_ptr()
    assert got["state"] % 16 == 0 and got["checkpoints"] % 16 == 0


@pytest.mark.parametrize("layout", ["padded", "packed"])
def test_borders_made_inside_a_checkpointed_block(library, layout):
    """The first pass's borders are gone when the backward pass runs: it has to read those of the second."""
    made = []

    def block(x, gate):
        if layout == "padded":
            made.append(torch.tensor([50, 7]).int())
            return ds.gated_recurrence(x, gate, lengths=made[-1])[0]
        made.append(torch.cumsum(torch.tensor([0, 40, 60]), 0).int())
        return ds.gated_recurrence(x, gate, offsets=made[-1])[0]

    shape = (2, 50, 8) if layout == "padded" else (100, 8)
    x, gate = torch.randn(shape, requires_grad=True), torch.randn(shape, requires_grad=True)
    h = checkpoint(block, x, gate, use_reentrant=False)
    torch.autograd.grad(h, [x, gate], torch.zeros_like(h))
    assert len(made) == 2
    assert library.backward[0]["offsets" if layout == "packed" else "lengths"] == made[1].data_ptr()


def test_two_backward_passes_of_one_graph_each_take_their_own_borders(library):
    x, gate = torch.randn(100, 8, requires_grad=True), torch.randn(100, 8, requires_grad=True)
    handed = []

    def hand_out(t):
        handed.append(anew(t))
        return handed[-1]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), hand_out):
        h, _ = ds.gated_recurrence(x, gate, offsets=torch.tensor([0, 40, 100], dtype=torch.int32))
    for _ in range(2):
        torch.autograd.grad(h, [x, gate], torch.zeros_like(h), retain_graph=True)
    seen = [b["offsets"] for b in library.backward]
    assert seen == [t.data_ptr() for t in handed if t.dtype == torch.int32] and seen[0] != seen[1]


@pytest.mark.parametrize("change", ["dtype", "rows", "checkpoints"])
def test_hooks_that_hand_out_something_else_are_refused(library, change):
    def hand_out(t):
        if change == "dtype" and t.shape == (100, 8):
            return t.half()
        if change == "rows" and t.shape == (100, 8):
            return t[:90]
        if change == "checkpoints" and t.dtype == torch.uint8:
            return t[:128]
        return t

    x, gate = torch.randn(100, 8, requires_grad=True), torch.randn(100, 8, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hand_out):
        h, _ = ds.gated_recurrence(x, gate, offsets=torch.tensor([0, 40, 100], dtype=torch.int32))
    with pytest.raises((RuntimeError, ValueError)):
        torch.autograd.grad(h, [x, gate], torch.zeros_like(h))
    assert not library.backward


# ---- on the GPU -------------------------------------------------------------------------------------------------------

def on_the_gpu(layout, d, heads, dtype, sliced, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    wide, gates = rand(3, 700, 2 * d).to(dtype), rand(3, 700, 2 * heads).to(dtype)
    x, gate = (wide[..., d:], gates[..., heads:]) if sliced else (wide[..., d:].contiguous(), gates[..., heads:].contiguous())
    if layout == "packed":
        x, gate = x.flatten(0, 1), gate.flatten(0, 1)
    lead = x.shape[:-1]
    return (x.requires_grad_(), gate.requires_grad_(), rand(3, d).requires_grad_()), (rand(*lead, d).to(dtype), rand(3, d))


def borders_of(layout):
    if layout == "padded":
        return dict(lengths=torch.tensor([700, 13, 400], device="cuda").int())
    if layout == "packed":
        return dict(offsets=torch.cumsum(torch.tensor([2, 900, 13, 1000], device="cuda"), 0).int())
    return {}


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["save_on_cpu", "anew", "spread_out", "checkpoint"])
@pytest.mark.parametrize("layout", ["dense", "padded", "packed"])
@pytest.mark.parametrize("sliced", [False, True])
@pytest.mark.parametrize("d, heads, dtype", [(64, 64, torch.bfloat16), (48, 3, torch.float32), (5, 5, torch.float16), (3, 3, torch.float32),
                                             (3, 1, torch.float32)])
def test_gradients_do_not_depend_on_where_saved_tensors_have_been(how, layout, sliced, d, heads, dtype):
    leaves, grads = on_the_gpu(layout, d, heads, dtype, sliced)

    def call(x, gate, state):
        return ds.gated_recurrence(x, gate, state, coupled=True, **borders_of(layout))      # borders that nobody else holds

    want_out = call(*leaves)
    want = torch.autograd.grad(want_out, leaves, grads)
    if how == "checkpoint":
        out = checkpoint(call, *leaves, use_reentrant=False)
    elif how == "save_on_cpu":
        with torch.autograd.graph.save_on_cpu():
            out = call(*leaves)
    else:
        unpack = anew if how == "anew" else spread_out
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: unpack(t)):
            out = call(*leaves)
    junk = [torch.full((n,), 1 << 30, dtype=torch.int32, device="cuda") for n in (3, 4, 128)]   # where freed borders may have lain
    got = torch.autograd.grad(out, leaves, grads)
    assert all(torch.equal(a, b) for a, b in zip(out, want_out))
    for name, a, b in zip(("dx", "dgate", "dstate"), got, want):
        assert torch.equal(a, b), name
    assert _capi.take_device_status() == 0 and junk


@pytest.mark.gpu
@pytest.mark.parametrize("pair", ["numbers", "tensor"])
def test_dropout_in_a_checkpointed_block_draws_the_same_mask_again(pair):
    """The block runs twice.  A pair that lives on the device is read both times: it is advanced after the backward pass."""
    x = torch.randn(2, 500, 32, device="cuda", requires_grad=True)
    gate = torch.randn(2, 500, 32, device="cuda", requires_grad=True)
    rng = (7, 9) if pair == "numbers" else torch.tensor([7, 9], dtype=torch.int64, device="cuda")
    v = torch.randn(2, 500, 32, device="cuda")

    def block(x, gate):
        h = ds.dropout(ds.gated_recurrence(x, gate, coupled=True)[0], 0.3, rng, residual=x)
        return h * torch.sigmoid(h)                        # its own backward pass takes the recomputed h

    want_out = block(x, gate)
    want = torch.autograd.grad(want_out, (x, gate), v)
    out = checkpoint(block, x, gate, use_reentrant=False)
    got = torch.autograd.grad(out, (x, gate), v)
    assert torch.equal(out, want_out) and all(torch.equal(a, b) for a, b in zip(got, want))
