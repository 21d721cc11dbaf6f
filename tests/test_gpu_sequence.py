"""Gated recurrence and dropout on the GPU, through the public entry points, against the float64 checker, and together with
the rasterizer: dropped splats composited by the recurrence are the rasterizer's image."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ds_splat_b200 as ds  # noqa: E402
from conftest import capi_camera, gradient_gate, scene_tensors, settings_for  # noqa: E402
from ds_splat_b200 import _capi, scenes  # noqa: E402
from ds_splat_b200.dp import CameraTensors, GradientBuffer, SplatDropout, ViewRenderer, data_parallel_step  # noqa: E402
from oracle import sequence_oracle as O  # noqa: E402

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
TINY = {"fp32": 1e-36, "fp16": 2.0 ** -25, "bf16": 1e-36}     # half a step of the smallest values; 32 bits flush denormals


def close(got, value, bound, dtype, what):
    """Within the checker's bound for 32-bit arithmetic (doubled: it is of first order, and the inputs of the second are the
    rounded results of the first) and half a step of the storage type."""
    got = got.detach().double().cpu().numpy()
    step = 0.0 if dtype == "fp32" else torch.finfo(DTYPES[dtype]).eps / 2
    limit = 2 * bound + step * (np.abs(value) + 2 * bound) + TINY[dtype]
    err = np.abs(got - value)
    assert np.isfinite(got).all(), what
    assert (err <= limit).all(), f"{what}: off by {(err / np.maximum(limit, 1e-300)).max():.2f} of the bound"


def make(n, d, heads, s, dtype, form, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    t = DTYPES[dtype]
    gate = (rand(n, heads) * 2 + 1) if form == "logit" else torch.rand((n, heads), generator=g, device="cuda") * 2 - 1
    return rand(n, d).to(t), gate.to(t), rand(s, d), rand(n, d).to(t), rand(s, d)


def check(layout, count, rows, d, heads, dtype="fp32", form="logit", coupled=False, reverse=False, final_only=False, state=True,
          begin=None, seed=1, outside_gate="inf"):
    """count: rows of every sequence; rows: rows of a dense or padded sequence, or of the packed tensor."""
    s = len(count)
    n = rows if layout == "packed" else rows * s
    if begin is None:
        begin = np.concatenate([[0], np.cumsum(count)])[:-1] if layout == "packed" else np.arange(s) * rows
    x, gate, st, v_h, v_last = make(n, d, heads, s, dtype, form, seed)
    more = {}
    if layout == "packed":
        more["offsets"] = torch.tensor(list(begin) + [begin[-1] + count[-1]] if s else [0], dtype=torch.int32, device="cuda")
    elif layout == "padded":
        more["lengths"] = torch.tensor(count, dtype=torch.int32, device="cuda")
    inside = np.zeros(n, bool)
    for b, c in zip(begin, count):
        inside[b:b + c] = True
    out = torch.from_numpy(~inside).cuda()
    want = O.recurrence(*(t.double().cpu().numpy() for t in (x, gate)), st.cpu().numpy() if state else np.zeros((s, d)), begin, count,
                        form, coupled, reverse, None if final_only else v_h.double().cpu().numpy(), v_last.cpu().numpy())
    # what lies in rows of no sequence must not matter
    x[out], gate[out], v_h[out] = float("nan"), float(outside_gate), float("nan")
    lead = (n,) if layout == "packed" else (s, rows)
    x, gate, v_h = (t.view(*lead, -1) for t in (x, gate, v_h))
    leaves = [x.requires_grad_(), gate.requires_grad_()] + ([st.requires_grad_()] if state else [])
    h, last = ds.gated_recurrence(x, gate, st if state else None, form=form, coupled=coupled, reverse=reverse, final_only=final_only, **more)
    assert (h is None) == final_only
    grads = torch.autograd.grad([last] if final_only else [h, last], leaves, [v_last] if final_only else [v_h, v_last])
    name = f"{layout} {count if s < 8 else s} {rows} {d}/{heads} {dtype} {form} {coupled} {reverse}"
    if not final_only:
        assert h.dtype == x.dtype and h.shape == x.shape
        close(h.reshape(n, d), *want["h"], dtype, name + " h")
        assert not h.reshape(n, d)[out].any()
    close(last, *want["last"], "fp32", name + " last")
    close(grads[0].reshape(n, d), *want["dx"], dtype, name + " dx")
    close(grads[1].reshape(n, heads), *want["dgate"], dtype, name + " dgate")
    assert not grads[0].reshape(n, d)[out].any() and not grads[1].reshape(n, heads)[out].any()
    if state:
        close(grads[2], *want["dstate"], "fp32", name + " dstate")
    with torch.no_grad():      # without a backward pass to come: the same values
        h2, last2 = ds.gated_recurrence(x, gate, st if state else None, form=form, coupled=coupled, reverse=reverse,
                                        final_only=final_only, **more)
    assert torch.equal(last2, last) and (final_only or torch.equal(h2, h))
    return h, last, grads


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 129, 1000])
@pytest.mark.parametrize("d", [128, 20, 3])
def test_lengths_around_the_tiles(rows, d):
    check("dense", [rows, rows], rows, d, d)
    check("dense", [rows, rows], rows, d, d, reverse=True, coupled=True, form="decay", dtype="bf16", state=False)


@pytest.mark.parametrize("d, heads", [(1, 1), (2, 2), (2, 1), (5, 5), (6, 2), (31, 1), (33, 33), (64, 1), (96, 8), (100, 100),
                                      (129, 129), (132, 132), (160, 1), (260, 2), (165, 5), (264, 1), (512, 4)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_channels_and_heads(d, heads, dtype):
    check("dense", [77] * 2, 77, d, heads, dtype=dtype, coupled=dtype != "fp16", form="logit" if dtype != "fp32" else "decay")
    check("packed", [30, 0, 1, 200, 7], 240, d, heads, dtype=dtype, coupled=dtype == "fp16", reverse=True)


@pytest.mark.parametrize("form", ["logit", "decay"])
@pytest.mark.parametrize("coupled", [False, True])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("final_only", [False, True])
def test_forms(form, coupled, reverse, final_only):
    for layout, count, rows in (("dense", [300, 300], 300), ("padded", [0, 5, 257, 300], 300), ("packed", [0, 0, 400, 1, 0, 90, 0], 500)):
        for d, heads in ((36, 36), (24, 3), (7, 1)):
            check(layout, count, rows, d, heads, form=form, coupled=coupled, reverse=reverse, final_only=final_only)


@pytest.mark.parametrize("reverse", [False, True])
def test_padded_batches_of_short_and_long_rows(reverse):
    check("padded", [0, 1, 2, 3, 0, 3], 3, 12, 12, reverse=reverse)                  # many sequences in one tile
    check("padded", [0] * 4, 9, 8, 8, reverse=reverse)                                 # nothing but padding
    check("padded", [700, 0, 1, 699], 700, 128, 128, dtype="fp16", reverse=reverse)    # whole tiles of padding
    check("padded", [5000 // 4] * 2, 1300, 4, 1, dtype="bf16", reverse=reverse)


@pytest.mark.parametrize("reverse", [False, True])
def test_packed_borders(reverse):
    check("packed", [1] * 300, 300, 8, 8, reverse=reverse)                           # every row a sequence of its own
    check("packed", [0] * 1000 + [40] + [0] * 1000, 64, 8, 8, reverse=reverse)       # borders that all lie on one row
    check("packed", [128, 128, 64, 64, 1, 127], 512, 64, 64, reverse=reverse)        # borders on the tiles' edges
    check("packed", [50, 60], 200, 16, 4, begin=[33, 83], reverse=reverse)           # rows before the first sequence
    check("packed", [3], 3000, 64, 64, reverse=reverse)                              # tiles without a sequence
    check("packed", [], 70, 8, 8, reverse=reverse)                                   # rows without a sequence


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("form", ["logit", "decay"])
def test_nan_gates_in_rows_of_no_sequence(form, reverse):
    for d, heads in ((12, 12), (12, 3), (7, 1), (3, 1), (3, 3)):
        check("padded", [0, 5, 90], 90, d, heads, form=form, reverse=reverse, coupled=True, outside_gate="nan")
        check("packed", [20, 30], 400, d, heads, form=form, reverse=reverse, begin=[40, 60], outside_gate="-inf")
        check("packed", [20, 30], 400, d, heads, form=form, reverse=reverse, begin=[40, 60], outside_gate="nan")


@pytest.mark.parametrize("reverse", [False, True])
def test_rows_of_three_channels(reverse):
    """32-bit rows of three channels are copied as one piece of memory: whole and partial tiles of 1280 rows, with and without
    borders, padding that covers tiles, several tiles per block, and rows that do not lie together."""
    kw = dict(reverse=reverse, coupled=True, form="decay")
    for heads in (1, 3):
        for rows in (1, 5, 1279, 1280, 1281, 4000):
            check("dense", [rows], rows, 3, heads, **kw)
        check("padded", [0, 1, 3000, 5000], 5000, 3, heads, **kw)
        check("packed", [1] * 3000, 3001, 3, heads, **kw)
        check("packed", [700, 0, 4000, 0, 0, 3, 1280, 1], 6500, 3, heads, final_only=True, **kw)
        check("packed", [300] * 9, 2800, 3, heads, state=False, **kw)
    wide = torch.randn(2, 2000, 8, device="cuda")
    gate = torch.rand(2, 2000, 1, device="cuda")
    a = ds.gated_recurrence(wide[..., 1:4], gate, reverse=reverse, form="decay")
    b = ds.gated_recurrence(wide[..., 1:4].contiguous(), gate, reverse=reverse, form="decay")
    for p, q in zip(a, b):      # two ways through the rows: sums of a few units, rounded in another order
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-4)
    x = wide[..., 1:4].contiguous().requires_grad_()
    h, _ = ds.gated_recurrence(x, gate, reverse=reverse, form="decay")
    v = torch.randn(2, 2000, 8, device="cuda")[..., 2:5]          # a gradient whose rows do not lie together
    got, = torch.autograd.grad(h, x, v, retain_graph=True)
    assert torch.equal(got, torch.autograd.grad(h, x, v.contiguous())[0])


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("d, heads, dtype", [(64, 64, "fp32"), (48, 3, "fp32"), (64, 1, "bf16"), (6, 6, "fp16"), (4, 1, "fp32"), (3, 1, "fp32"), (1, 1, "bf16")])
def test_many_tiles_and_segments(d, heads, dtype, reverse):
    """Long enough to be cut into segments whose maps are carried on: one sequence, a few whose borders lie anywhere, and a padded
    batch; the composition passes segments with and without borders."""
    check("dense", [12000], 12000, d, heads, dtype=dtype, reverse=reverse, coupled=True)
    check("packed", [1, 5000, 0, 40, 40, 1, 6800, 13], 12000, d, heads, dtype=dtype, reverse=reverse)
    check("padded", [0, 4000, 37], 4000, d, heads, dtype=dtype, reverse=reverse)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [148, 160, 192, 204, 256])
def test_only_the_last_state_of_long_wide_rows(d, dtype):
    """Segments without an output: the backward pass over them holds just under 31 KB beside its static shared memory."""
    for reverse in (False, True):
        check("dense", [9000], 9000, d, d, dtype=dtype, final_only=True, reverse=reverse)
        check("packed", [1, 4000, 0, 40, 4959], 9000, d, d, dtype=dtype, final_only=True, reverse=reverse)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("d, heads", [(10, 5), (18, 9), (21, 7), (78, 26), (99, 33), (35, 7), (36, 3), (80, 5), (68, 17), (14, 2), (108, 9)])
def test_many_narrow_heads(d, heads, dtype):
    """Several heads in a block, the last block's not all there; cut into segments and not."""
    for reverse in (False, True):
        kw = dict(dtype=dtype, reverse=reverse, coupled=dtype == "bf16", form="decay" if reverse else "logit")
        check("dense", [90] * 2, 90, d, heads, **kw)
        check("dense", [7000], 7000, d, heads, **kw)
        check("packed", [1, 3000, 0, 0, 40, 1, 800, 13], 3900, d, heads, outside_gate="nan", **kw)
        check("padded", [0, 2500, 37, 1], 2500, d, heads, outside_gate="nan", **kw)
        check("packed", [1] * 400 + [0] * 300 + [200], 700, d, heads, final_only=True, **kw)


def test_more_borders_in_a_tile_than_threads_look_at_once():
    for reverse in (False, True):
        check("packed", [1] * 2500, 2600, 1, 1, reverse=reverse)
        check("packed", [0, 1, 0] * 700, 700, 3, 1, reverse=reverse, coupled=True)
        check("packed", [0] * 255 + [1] + [0] * 600 + [2], 9, 8, 8, reverse=reverse)
        check("dense", [1] * 2500, 1, 4, 4, reverse=reverse)
        check("padded", [1, 0] * 900, 2, 1, 1, reverse=reverse)


def test_no_rows_and_no_sequences():
    st = torch.randn(3, 8, device="cuda", requires_grad=True)
    x = torch.zeros(3, 0, 8, device="cuda", requires_grad=True)
    h, last = ds.gated_recurrence(x, x.detach(), st)
    assert h.shape == (3, 0, 8) and torch.equal(last, st)
    dx, dst = torch.autograd.grad(last, (x, st), torch.ones_like(last))
    assert dx.shape == x.shape and torch.equal(dst, torch.ones_like(st))
    h, last = ds.gated_recurrence(x, x.detach(), st, lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert h.shape == (3, 0, 8) and torch.equal(last, st)
    h, last = ds.gated_recurrence(torch.zeros(0, 5, 8, device="cuda"), torch.zeros(0, 5, 8, device="cuda"))
    assert h.shape == (0, 5, 8) and last.shape == (0, 8)
    h, last = ds.gated_recurrence(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 1, device="cuda"),
                                  offsets=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert h.shape == (0, 8) and last.shape == (0, 8)
    h, last = ds.gated_recurrence(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 1, device="cuda"), torch.ones(2, 8, device="cuda"),
                                  offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert torch.equal(last, torch.ones(2, 8, device="cuda"))
    assert ds.gated_recurrence_step(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 8, device="cuda"),
                                    torch.zeros(0, 8, device="cuda")).shape == (0, 8)


def test_gates_that_open_and_close_entirely_and_infinities_that_stay_in_their_sequence():
    x = torch.randn(4, 300, 16, device="cuda")
    g = torch.randn(4, 300, 16, device="cuda")
    g[:, 100] = float("-inf")          # everything before is forgotten
    g[:, 200:] = float("inf")          # everything is kept, coupled nothing comes in
    h, last = ds.gated_recurrence(x, g, coupled=True)
    assert torch.equal(h[:, 100], x[:, 100])
    want = O.recurrence(x.double().cpu().numpy().reshape(-1, 16), g.double().cpu().numpy().reshape(-1, 16), np.zeros((4, 16)),
                        np.arange(4) * 300, [300] * 4, "logit", True, False)
    close(h.reshape(-1, 16), *want["h"], "fp32", "h")
    close(last, *want["last"], "fp32", "last")
    x[1, 50, 3] = float("inf")         # one sequence, one channel; its row 100 forgets 0 * inf into NaN
    x[2, 7] = float("nan")
    for kw in (dict(), dict(reverse=True)):
        clean, _ = ds.gated_recurrence(torch.nan_to_num(x, 0.0, 0.0), g, **kw)
        got, _ = ds.gated_recurrence(x, g, **kw)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[3], clean[3])
        same = torch.ones(16, dtype=torch.bool, device="cuda")
        same[3] = False
        assert torch.equal(got[1][:, same], clean[1][:, same])
        flat = ds.gated_recurrence(x.view(-1, 16), g.view(-1, 16), offsets=torch.arange(0, 1201, 300, dtype=torch.int32, device="cuda"), **kw)[0]
        for s in (0, 3):               # magnitudes of a few units, a bound of 2 * 16 u per row that a gate's decay leaves
            torch.testing.assert_close(flat.view_as(x)[s], clean[s], rtol=1e-5, atol=1e-5)


def test_strides_alignments_and_broadcast_inputs():
    wide = torch.randn(3, 50, 2 * 24, device="cuda")
    gates = torch.randn(3, 50, 24, device="cuda")
    want = ds.gated_recurrence(wide[..., 24:].contiguous(), gates)
    for x in (wide[..., 24:], torch.randn(1 + 3 * 50 * 24, device="cuda")[1:].view(3, 50, 24).copy_(wide[..., 24:]),
              wide[..., 24:].transpose(0, 1).contiguous().transpose(0, 1)):
        for g in (gates, torch.cat([gates, gates], -1)[..., 24:]):
            got = ds.gated_recurrence(x, g)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a gradient that arrives broadcast (a sum's), and inputs that are broadcast: their gradients sum
    x1 = torch.randn(24, device="cuda", requires_grad=True)
    g1 = torch.randn(50, 24, device="cuda", requires_grad=True)
    st = torch.randn(24, device="cuda", requires_grad=True)
    h, last = ds.gated_recurrence(x1.expand(3, 50, 24), g1.expand(3, 50, 24), st.expand(3, 24))
    (h.sum() + last.sum()).backward()
    x2, g2, s2 = (t.detach().double().cpu().numpy() for t in (x1, g1, st))
    w = O.recurrence(np.tile(x2, (150, 1)), np.tile(g2, (3, 1)), np.tile(s2, (3, 1)), [0, 50, 100], [50] * 3, "logit", False, False,
                     np.ones((150, 24)), np.ones((3, 24)))
    sums = lambda v, *s: v.reshape(*s).sum(tuple(range(len(s) - 1))) if len(s) > 1 else v  # noqa: E731
    # torch adds the copies in 32 bits: at most one rounding of the running sum of magnitudes per copy
    for t, (v, b), copies, shape in ((x1, w["dx"], 150, (150, 24)), (st, w["dstate"], 3, (3, 24))):
        close(t.grad, sums(v, *shape), sums(b, *shape) + copies * O.U * sums(np.abs(v), *shape), "fp32", "broadcast")
    v, b = w["dgate"]
    close(g1.grad, v.reshape(3, 50, 24).sum(0), b.reshape(3, 50, 24).sum(0) + 3 * O.U * np.abs(v).reshape(3, 50, 24).sum(0), "fp32", "gate")


def test_only_some_gradients_are_asked_for():
    x, g, st, v_h, v_last = make(2 * 90, 32, 32, 2, "fp32", "logit", 5)
    x, g, v_h = (t.view(2, 90, 32) for t in (x, g, v_h))
    full = torch.autograd.grad(ds.gated_recurrence(x.requires_grad_(), g.requires_grad_(), st.requires_grad_()), (x, g, st), (v_h, v_last))
    for k in range(3):
        args = [t.detach().clone() for t in (x, g, st)]
        args[k].requires_grad_()
        got, = torch.autograd.grad(ds.gated_recurrence(*args), args[k], (v_h, v_last))
        assert torch.equal(got, full[k])
    h, last = ds.gated_recurrence(x, g, st)          # one output alone takes part in the loss
    a = torch.autograd.grad(h, (x, g, st), v_h, retain_graph=True)
    b = torch.autograd.grad(last, (x, g, st), v_last)
    z = torch.autograd.grad(ds.gated_recurrence(x, g, st), (x, g, st), (v_h, torch.zeros_like(v_last)))
    assert all(torch.equal(p, q) for p, q in zip(a, z))
    z = torch.autograd.grad(ds.gated_recurrence(x, g, st), (x, g, st), (torch.zeros_like(v_h), v_last))
    assert all(torch.equal(p, q) for p, q in zip(b, z))


def test_gradient_against_differences_on_the_device():
    """Along one direction per input, in fp32: the central difference of the loss against the gradient's product."""
    x, g, st, v_h, v_last = make(3 * 40, 12, 4, 3, "fp32", "logit", 6)
    x, g, v_h = x.view(3, 40, 12), g.view(3, 40, 4), v_h.view(3, 40, 12)
    args = [t.requires_grad_() for t in (x, g, st)]
    grads = torch.autograd.grad(ds.gated_recurrence(*args, coupled=True), args, (v_h, v_last))

    def loss(*a):
        h, last = ds.gated_recurrence(*a, coupled=True)
        return float((h.double() * v_h.double()).sum() + (last.double() * v_last.double()).sum()), \
            float((h.double() * v_h.double()).abs().sum() + (last.double() * v_last.double()).abs().sum())

    step = 2.0 ** -7
    with torch.no_grad():
        for k, a in enumerate(args):
            way = torch.randn_like(a).sign()
            moved = lambda sign: [t + sign * step * way if i == k else t for i, t in enumerate(args)]  # noqa: E731
            (up, size), (down, _) = loss(*moved(1)), loss(*moved(-1))
            slope = (up - down) / (2 * step)
            want = float((grads[k].double() * way.double()).sum())
            # rounding: both losses within 2 * 40 rows' bounds of u; the step's own error is third order, under step^2 of the
            # sum of magnitudes
            assert abs(slope - want) <= size * (2 * 40 * O.ROW * O.U / step + step * step), k


def test_step_is_the_recurrence_one_row_at_a_time():
    for dtype, d, heads, form, coupled in (("bf16", 64, 64, "logit", True), ("fp16", 48, 3, "decay", False), ("fp32", 7, 7, "logit", False),
                                           ("bf16", 9, 3, "decay", True), ("fp32", 5, 1, "logit", True)):
        x, g, st, _, _ = make(6 * 5, d, heads, 6, dtype, form, 7)
        x, g = x.view(6, 5, d), g.view(6, 5, heads)
        h, last = ds.gated_recurrence(x, g, st, form=form, coupled=coupled)
        state = st.clone()
        version = state._version
        for t in range(5):
            got = ds.gated_recurrence_step(x[:, t], g[:, t], state, form=form, coupled=coupled)
            n = x.shape[0]
            want = O.recurrence(x[:, :t + 1].double().cpu().numpy().reshape(-1, d), g[:, :t + 1].double().cpu().numpy().reshape(-1, heads),
                                st.cpu().numpy(), np.arange(n) * (t + 1), [t + 1] * n, form, coupled, False)
            close(got, want["h"][0].reshape(n, t + 1, d)[:, -1], want["h"][1].reshape(n, t + 1, d)[:, -1], dtype, "step h")
            close(state, *want["last"], "fp32", "step state")
        assert state._version > version


def test_refusals_on_the_device():
    x, g = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 3, 8, device="cuda")
    offsets = torch.zeros(3, dtype=torch.int32, device="cuda")
    bad = [
        (RuntimeError, lambda: ds.gated_recurrence(x.double(), g.double())), (RuntimeError, lambda: ds.gated_recurrence(x, g.half())),
        (RuntimeError, lambda: ds.gated_recurrence(x, g.cpu())), (ValueError, lambda: ds.gated_recurrence(x, g[:, :2])),
        (ValueError, lambda: ds.gated_recurrence(x, g[..., :3])), (ValueError, lambda: ds.gated_recurrence(x[0], g[0])),
        (ValueError, lambda: ds.gated_recurrence(x, g, form="sigmoid")), (ValueError, lambda: ds.gated_recurrence(x, g, offsets=offsets)),
        (ValueError, lambda: ds.gated_recurrence(x[0], g[0], offsets=offsets, lengths=offsets)),
        (RuntimeError, lambda: ds.gated_recurrence(x[0], g[0], offsets=offsets.long())),
        (RuntimeError, lambda: ds.gated_recurrence(x[0], g[0], offsets=offsets.cpu())),
        (ValueError, lambda: ds.gated_recurrence(x[0], g[0], offsets=offsets[:0])),
        (ValueError, lambda: ds.gated_recurrence(x, g, lengths=offsets)),
        (RuntimeError, lambda: ds.gated_recurrence(x, g, torch.zeros(2, 8, device="cuda", dtype=torch.float16))),
        (ValueError, lambda: ds.gated_recurrence(x, g, torch.zeros(3, 8, device="cuda"))),
        (ValueError, lambda: ds.gated_recurrence_step(x, g, x)), (ValueError, lambda: ds.gated_recurrence_step(x[0], g[0], x[0, :2])),
        (ValueError, lambda: ds.gated_recurrence_step(x[0, :, :4], g[0, :, :4], x[0, :, :4])),
        (RuntimeError, lambda: ds.gated_recurrence_step(x[0].half(), g[0].half(), x[0].half())),
        (RuntimeError, lambda: ds.gated_recurrence_step(x[0].clone().requires_grad_(), g[0], x[0].clone())),
        (ValueError, lambda: ds.dropout(x, 1.5, (0, 0))), (ValueError, lambda: ds.dropout(x, float("nan"), (0, 0))),
        (ValueError, lambda: ds.dropout(x, 0.5, (-1, 0))), (ValueError, lambda: ds.dropout(x, 0.5, (0, 1 << 64))),
        (ValueError, lambda: ds.dropout(x, 0.5, (0, 0), residual=x[0])), (RuntimeError, lambda: ds.dropout(x, 0.5, (0, 0), residual=x.half())),
        (RuntimeError, lambda: ds.dropout(x.double(), 0.5, (0, 0))), (RuntimeError, lambda: ds.dropout(x, 0.5, torch.zeros(2, device="cuda"))),
        (ValueError, lambda: ds.dropout(x, 0.5, torch.zeros(3, dtype=torch.int64, device="cuda"))),
        (RuntimeError, lambda: ds.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


@pytest.mark.parametrize("values", [[0, 5, 3, 10], [0, 4, 8, 64], [-3, 2, 4, 10], [2, 1, 0, 0]])
def test_offsets_out_of_order_or_range_are_reported(values):
    """Every access stays within the tensors whatever the offsets say (reasoned for the kernels' index arithmetic); the status
    word tells."""
    x = torch.randn(10, 8, device="cuda", requires_grad=True)
    offsets = torch.tensor(values, dtype=torch.int32, device="cuda")
    _capi.take_device_status()
    _, last = ds.gated_recurrence(x, torch.randn(10, 8, device="cuda"), offsets=offsets)
    with pytest.raises(_capi.DsbError) as info:
        _capi.take_device_status()
    assert info.value.code == -1 and "offsets" in str(info.value)
    assert _capi.take_device_status() == 0
    torch.autograd.grad(last, x, torch.ones_like(last))
    with pytest.raises(_capi.DsbError):
        _capi.take_device_status()
    y = torch.randn(3, 10, 8, device="cuda")
    ds.gated_recurrence(y, y, lengths=torch.tensor([1, 11, 2], dtype=torch.int32, device="cuda"))
    with pytest.raises(_capi.DsbError):
        _capi.take_device_status()
    assert _capi.take_device_status() == 0


def test_the_same_call_gives_the_same_bits_on_any_stream_and_in_a_replayed_graph():
    x, g, st, v_h, v_last = make(40000, 64, 8, 5, "bf16", "logit", 8)
    offsets = torch.tensor([0, 10, 9000, 9000, 25000, 39999], dtype=torch.int32, device="cuda")
    leaves = [x.requires_grad_(), g.requires_grad_(), st.requires_grad_()]

    def step():
        h, last = ds.gated_recurrence(x, g, st, offsets=offsets)
        grads = torch.autograd.grad((h, last), leaves, (v_h, v_last))
        return [h.detach(), last.detach(), *grads]

    want = step()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                               # two graphs, replayed beside each other
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for _ in range(3):
        for (graph, out), s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                for t in out:
                    t.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    with torch.no_grad():                            # new inputs in the same place reach the replayed graph
        x.mul_(0.5)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], step()))


def test_elements_past_two_to_the_31():
    """A packed tensor whose last sequence lies past 2^31 elements: its values come from the right place."""
    rows, d, tail = (1 << 21) + 77, 1024, 50
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    gate = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    xs, gs, _, vs, v_last = make(tail, d, d, 2, "bf16", "logit", 9)
    x[-tail:], gate[-tail:] = xs, gs
    offsets = torch.tensor([0, rows - tail, rows], dtype=torch.int32, device="cuda")
    x.requires_grad_()
    h, last = ds.gated_recurrence(x, gate, offsets=offsets)
    v_h = torch.zeros_like(h)
    v_h[-tail:] = vs
    dx, = torch.autograd.grad((h, last), x, (v_h, v_last))
    w = O.recurrence(xs.double().cpu().numpy(), gs.double().cpu().numpy(), np.zeros((1, d)), [0], [tail], "logit", False, False,
                     vs.double().cpu().numpy(), v_last[1:].cpu().numpy())
    close(h[-tail:], *w["h"], "bf16", "h")
    close(last[1:], *w["last"], "fp32", "last")
    close(dx[-tail:], *w["dx"], "bf16", "dx")
    assert not h[:-tail].any() and not last[0].any()


# ---- dropout -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (7, 5), (129, 1023), (64, 256), (2, 3, 8), (100003,)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_against_the_checker(shape, dtype, residual):
    t = DTYPES[dtype]
    x = torch.randn(shape, device="cuda").to(t).requires_grad_()
    r = torch.randn(shape, device="cuda").to(t).requires_grad_() if residual else None
    for p, rng in ((0.3, (12345678901234567890, 7)), (0.0, (1, 2)), (1.0, (1, 2)), (0.999, (0, (1 << 64) - 1))):
        out = ds.dropout(x, p, rng, residual=r)
        value, keep = O.dropout(x.detach().double().cpu().numpy(), p, *rng, r.detach().double().cpu().numpy() if residual else None)
        part = np.where(keep, np.abs(x.detach().double().cpu().numpy()) / max(1 - p, 1e-300), 0.0) if p < 1 else np.zeros(shape)
        # the scale is rounded to 32 bits, the fused product and sum once more: u of each
        close(out, value, O.U * part + O.U * np.abs(value), dtype, "dropout")
        v = torch.randn(shape, device="cuda").to(t)
        grads = torch.autograd.grad(out, (x, r) if residual else (x,), v)
        vn = v.double().cpu().numpy()
        want, _ = O.dropout(vn, p, *rng)
        close(grads[0], want, 2 * O.U * np.abs(want), dtype, "dropout's gradient")
        assert np.array_equal(grads[0].cpu().double().numpy() != 0, keep & (vn != 0) & (p < 1))
        if residual:
            assert torch.equal(grads[1], v)


def test_dropout_does_not_depend_on_how_a_tensor_lies():
    x = torch.randn(6, 37, 24, device="cuda").half()
    r = torch.randn(6, 37, 24, device="cuda").half()
    want, want_r = ds.dropout(x, 0.4, (3, 4)), ds.dropout(x, 0.4, (3, 4), residual=r)
    pad = lambda t: torch.cat([t, t], -1)[..., 24:]  # noqa: E731
    off = torch.empty(6 * 37 * 24 + 1, device="cuda", dtype=torch.float16)[1:].view(6, 37, 24)
    off.copy_(x)
    for y in (pad(x), off, x.transpose(0, 1).contiguous().transpose(0, 1), pad(x)[:, :, :]):
        assert torch.equal(ds.dropout(y, 0.4, (3, 4)), want)
        for s in (r, pad(r)):
            assert torch.equal(ds.dropout(y, 0.4, (3, 4), residual=s), want_r)
    one = torch.randn(24, device="cuda").half()
    assert torch.equal(ds.dropout(one.expand(5, 24), 0.4, (3, 4)), ds.dropout(one.expand(5, 24).contiguous(), 0.4, (3, 4)))
    leaf = torch.randn(5, 24, device="cuda").requires_grad_()
    ds.dropout(leaf, 0.4, (3, 4)).sum().backward()           # a broadcast gradient
    assert torch.equal(leaf.grad, ds.dropout(torch.ones(5, 24, device="cuda"), 0.4, (3, 4)))
    assert ds.dropout(torch.zeros(0, 3, device="cuda"), 0.5, (0, 0)).shape == (0, 3)
    assert ds.dropout(torch.ones((), device="cuda"), 0.0, (0, 0)) == 1


def test_dropped_places_leave_no_trace_of_infinities_and_nan():
    x = torch.ones(4096, device="cuda")
    keep = ds.dropout(x, 0.5, (5, 6)) != 0
    x[~keep] = float("nan")
    x[(~keep).nonzero()[::2, 0]] = float("inf")
    assert torch.equal(ds.dropout(x, 0.5, (5, 6)), keep.float() * 2)
    assert torch.equal(ds.dropout(x, 0.5, (5, 6), residual=torch.ones_like(x)), keep.float() * 2 + 1)
    full = torch.full((64,), float("inf"), device="cuda")
    assert not ds.dropout(full, 1.0, (5, 6)).any()


def test_share_of_kept_elements_and_independence_of_steps():
    n = 1 << 20
    x = torch.ones(n, device="cuda")
    for p in (0.01, 0.5, 0.9):
        a, b = (ds.dropout(x, p, (17, s)) != 0 for s in (0, 1))
        c = ds.dropout(x, p, (18, 0)) != 0
        spread = 6 * (n * p * (1 - p)) ** 0.5           # six standard deviations
        assert abs(float(a.sum()) - n * (1 - p)) < spread
        for other in (b, c):
            q = (1 - p) ** 2
            assert abs(float((a & other).sum()) - n * q) < 6 * (n * q * (1 - q)) ** 0.5


def test_generator_state_on_the_device():
    x = torch.randn(1000, device="cuda", requires_grad=True)
    rng = torch.tensor([99, 5], dtype=torch.int64, device="cuda")
    out = ds.dropout(x, 0.3, rng)
    rng[1] += 1                                              # advanced before the backward pass: the old mask holds
    grad, = torch.autograd.grad(out, x, torch.ones_like(out))
    out = out.detach()          # torch captures a backward pass only while no eager graph of the same leaves lives
    assert torch.equal(out, ds.dropout(x, 0.3, (99, 5)))
    assert torch.equal(grad, ds.dropout(torch.ones_like(x), 0.3, (99, 5)))
    big = torch.tensor([-1, -2], dtype=torch.int64, device="cuda")   # the same bits as 2^64 - 1 and 2^64 - 2
    assert torch.equal(ds.dropout(x, 0.3, big), ds.dropout(x, 0.3, ((1 << 64) - 1, (1 << 64) - 2)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ds.dropout(x, 0.3, rng)
        g, = torch.autograd.grad(y, x, torch.ones_like(y))
        rng[1] += 1
    for step in (6, 7, 8):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ds.dropout(x, 0.3, (99, step)))
        assert torch.equal(g, ds.dropout(torch.ones_like(x), 0.3, (99, step)))


# ---- together, and with the rasterizer --------------------------------------------------------------------------------

def pixel_lists(records, pairs, ranges, h, w):
    """Every pixel's depth-ordered list, packed: alpha / opacity of each entry (0 where the blend skips it), splat ids, offsets."""
    tiles_x = (w + 15) // 16
    weights, ids, count = [], [], []
    for y in range(h):
        for x in range(w):
            t = (y // 16) * tiles_x + x // 16
            i = (pairs[int(ranges[t]):int(ranges[t + 1])] & 0xFFFFFFFF).long()
            q = records[i]
            dx, dy = q[:, 0] - (x + 0.5), q[:, 1] - (y + 0.5)
            power = -0.5 * (q[:, 2] * dx * dx + q[:, 4] * dy * dy) - q[:, 3] * dx * dy
            vis = torch.exp(power)
            seen = (power < 0) & (q[:, 5] * vis >= 1 / 255)
            weights.append(torch.where(seen, vis, torch.zeros_like(vis)))
            ids.append(i)
            count.append(len(i))
    return torch.cat(weights), torch.cat(ids), np.concatenate([[0], np.cumsum(count)]).astype(np.int32)


def test_dropped_splats_composited_by_the_recurrence_are_the_rasterizers_image():
    """dropout of the opacities -> the rasterizer, against dropout -> per-pixel lists -> gated recurrence back to front:
    the image, and the opacities' and colours' gradients through either."""
    sc = scenes.tiny(n=120, seed=41, W=32, H=32, focal=30.0)
    t = scene_tensors(sc)
    view, h, w = sc.views[0], sc.views[0].H, sc.views[0].W
    rng, p = (2024, 3), 0.25
    raw = (t["opacities"].clamp(0.05, 0.6)).detach()
    colors = torch.rand(sc.n, 3, device="cuda")
    v_image = torch.randn(h, w, 3, device="cuda")

    a_op, a_col = raw.clone().requires_grad_(), colors.clone().requires_grad_()
    dropped = ds.dropout(a_op, p, rng)
    image, radii = ds.GaussianRasterizer(settings_for(view, strict_reference=False))(
        t["means"], torch.zeros_like(t["means"]), None, a_col, dropped, t["scales"], t["rotations"], None)
    image.backward(v_image)

    cam, keep = capi_camera(view, drop_last=False)
    records, _, tiles, cov, keys = _capi.preprocess(cam, t["means"], None, dropped.detach(), t["scales"], t["rotations"], colors_precomp=colors)
    offsets, k = _capi.plan_pairs(cam, tiles, keys)
    pairs = _capi.sort_pairs(_capi.emit_pairs(cam, k, records, tiles, keys, offsets), 32, 40)
    ranges = _capi.identify_tile_ranges(pairs, h, w)
    weights, ids, lists = pixel_lists(records, pairs, ranges, h, w)
    b_op, b_col = raw.clone().requires_grad_(), colors.clone().requires_grad_()
    alphas = ds.dropout(b_op, p, rng).view(-1)[ids] * weights
    assert float(alphas.detach().max()) < 0.99          # below the blend's clamps
    _, pixels = ds.gated_recurrence(b_col[ids], 1 - alphas[:, None], offsets=torch.from_numpy(lists).cuda(), form="decay",
                                    coupled=True, reverse=True, final_only=True)
    pixels.view(h, w, 3).backward(v_image)

    # The blend stops where 1e-4 of the light is left: at most that much colour (below 1) is missing.  Both sides round
    # and take approximate exponentials besides.
    assert float((pixels.view(h, w, 3) - image).abs().max()) < 2e-4
    assert int((b_op.grad == 0).sum()) >= int((ds.dropout(raw, p, rng) == 0).sum()) > 0
    for name, got, want in (("opacities", b_op.grad, a_op.grad), ("colours", b_col.grad, a_col.grad)):
        err = (got - want).abs().max() / want.abs().max()
        assert float(err) < 2e-3, (name, float(err))


@pytest.mark.parametrize("accumulate", [False, True])
def test_training_step_with_dropped_splats(accumulate):
    """render_views with a dropout against a renderer of the opacities that ``dropout`` returns, its gradients taken back."""
    sc = scenes.headline(n=15_000, seed=92, W=256, H=160, focal=180.0, views=10, ring=True)
    t = scene_tensors(sc)
    cams = [CameraTensors.from_view(v, "cuda") for v in sc.views]
    vimgs = [torch.from_numpy(sc.image_grad(i)).cuda() for i in range(len(sc.views))]
    drop = SplatDropout(0.3, seed=77, step=12)
    renderer = ViewRenderer(t["means"], t["shs"], t["opacities"], t["scales"], t["rotations"])
    before = t["opacities"].clone()
    got = GradientBuffer(sc.n, "cuda")
    got.flat.fill_(3.0)
    if accumulate:
        renderer.render_views(cams[:3], vimgs[:3], got)      # something of the same size to add to
    base = {key: v.clone() for key, v in got.views.items()}
    renderer.render_views(cams, vimgs, got, accumulate=accumulate, dropout=drop)
    assert torch.equal(t["opacities"], before)
    leaf = t["opacities"].clone().requires_grad_()
    dropped = ds.dropout(leaf, drop.p, (drop.seed, drop.step))
    plain = ViewRenderer(t["means"], t["shs"], dropped.detach(), t["scales"], t["rotations"])
    want = GradientBuffer(sc.n, "cuda")
    want.flat.fill_(3.0)
    plain.render_views(cams, vimgs, want, accumulate=False)
    v_op, = torch.autograd.grad(dropped, leaf, want.views["opacities"].view_as(leaf))
    want.views["opacities"].copy_(v_op.view_as(want.views["opacities"]))
    for key in ("means3d", "shs", "opacities", "scales", "rotations"):
        a = got.views[key] - base[key] if accumulate else got.views[key]
        gradient_gate(a.cpu().numpy(), want.views[key].cpu().numpy(), key)
    gone = (dropped == 0).view(-1)
    left = base["opacities"].view(-1)[gone] if accumulate else torch.zeros(int(gone.sum()), device="cuda")
    assert torch.equal(got.views["opacities"].view(-1)[gone], left)
    # every splat dropped: nothing is drawn, and the gradients are zero
    none = GradientBuffer(sc.n, "cuda")
    images = []
    renderer.render_views(cams[:2], lambda i, image: (images.append(float(image.abs().max())), vimgs[i])[1], none, dropout=SplatDropout(1.0, 1))
    assert images == [0.0, 0.0] and not none.views["opacities"].any() and not none.views["shs"].any()
    # the data-parallel step hands the argument on, and without it nothing changes
    again = GradientBuffer(sc.n, "cuda")
    data_parallel_step(renderer, cams, vimgs, again, dropout=drop)
    assert bool((again.views["opacities"].view(-1)[gone] == 0).all())
    data_parallel_step(renderer, cams, vimgs, again)
    assert bool((again.views["opacities"].view(-1)[gone] != 0).any())


def test_calls_on_two_streams_at_once():
    """Calls that overlap share nothing: workspaces, border tables and checkpoints are each call's own."""
    inputs = [make(20000, 64, 16, 3, "bf16", "logit", 20 + i) for i in range(2)]
    offsets = torch.tensor([0, 7000, 7001, 20000], dtype=torch.int32, device="cuda")

    def run(x, g, st, v_h, v_last):
        leaves = [t.detach().requires_grad_() for t in (x, g, st)]
        h, last = ds.gated_recurrence(*leaves, offsets=offsets, coupled=True)
        return [h.detach(), last.detach(), *torch.autograd.grad((h, last), leaves, (v_h, v_last))]

    want = [run(*i) for i in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(run(*inputs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))


def test_changed_inputs_are_noticed_before_the_backward_pass():
    x = torch.randn(2, 30, 8, device="cuda", requires_grad=True)
    g = torch.randn(2, 30, 8, device="cuda")
    lengths = torch.tensor([30, 4], dtype=torch.int32, device="cuda")
    h, _ = ds.gated_recurrence(x, g, lengths=lengths)
    lengths[1] = 9
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    h, _ = ds.gated_recurrence(x, g)
    g.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def test_gradients_of_gradients_are_refused():
    x = torch.randn(1, 9, 4, device="cuda", requires_grad=True)
    h, _ = ds.gated_recurrence(x, x)
    first, = torch.autograd.grad(h.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), x)
    y = ds.dropout(x, 0.5, (1, 1))
    first, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), x)
