"""Cases of the sequence operators: the gated recurrence (whole sequences, training, single tokens) and dropout.

``own`` selects what ``run`` does: the framework's operators (True) or their plain form in elementary torch
operations (False).  Both take the same inputs and return the same outputs.

    recurrence   f_t = gate_t or sigmoid(gate_t);  h_t = f_t h_{t-1} + (x_t  or, coupled, (1 - f_t) x_t)
    dropout      out_i = [residual_i +] (x_i / (1 - p) where word i of Philox4x32-10 is at least p 2^32, else 0)
"""
import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def recurrence(name, **kw):
    case = dict(name=name, op="recurrence", layout="dense", batch=1, rows=1, channels=1, heads=0, dtype="bf16", form="logit",
                coupled=True, reverse=False, train=True, final_only=False, longest=0)
    case.update(kw)
    case["heads"] = case["heads"] or case["channels"]          # a gate value per channel unless told otherwise
    case["longest"] = case["longest"] or case["rows"]
    return case


def listed():
    return [
        # one token for a few sequences: latency alone
        dict(name="step_few", op="step", batch=4, channels=1024, heads=1024, dtype="bf16", form="logit", coupled=True),
        # one token for a full serving batch, one decay per head of 64 channels
        dict(name="step_batch", op="step", batch=768, channels=4096, heads=64, dtype="fp16", form="decay", coupled=False),
        # taking in a padded batch of prompts: forward only, odd lengths, state kept for the tokens to come
        recurrence("prompts_padded", layout="padded", batch=24, rows=1531, channels=1280, train=False),
        # a training step of a narrow layer in full precision, nothing a multiple of anything
        recurrence("train_odd_fp32", batch=5, rows=1001, channels=333, dtype="fp32", coupled=False),
        # the ordinary training step of a wide layer
        recurrence("train_wide", batch=8, rows=4096, channels=2560),
        # packed sequences of very different lengths, one decay per head: its gradient sums over the head's channels
        recurrence("train_packed_heads", layout="packed", batch=61, rows=30011, longest=9000, channels=1024, heads=16,
                   form="decay", coupled=False),
        # one sequence as long as a splat cloud is ordered, few channels: nothing but the sequence to split
        recurrence("train_long_narrow", batch=1, rows=131071, channels=64, dtype="fp32"),
        # compositing depth-ordered lists of colours back to front, one list per pixel: 1 - alpha is the list's shared decay,
        # only the composited pixel is wanted
        recurrence("composite_pixels", layout="packed", batch=115200, rows=4000037, longest=640, channels=3, heads=1,
                   dtype="fp32", form="decay", coupled=True, reverse=True, final_only=True),
        # compositing a wider feature vector for fewer pixels
        recurrence("composite_features", layout="packed", batch=9000, rows=330007, longest=512, channels=32, heads=1,
                   dtype="fp16", form="decay", coupled=True, reverse=True, final_only=True),
        # opacities of a 1M-splat cloud, dropped per splat
        dict(name="drop_opacities", op="dropout", rows=1000000, cols=1, dtype="fp32", p=0.2, residual=False),
        # a layer's output dropped and added to its residual stream
        dict(name="drop_residual", op="dropout", rows=32768, cols=2560, dtype="bf16", p=0.1, residual=True),
        # a small odd tensor: latency
        dict(name="drop_small_odd", op="dropout", rows=129, cols=1023, dtype="fp16", p=0.5, residual=False),
    ]


def spread(rng, low, high):
    """A size whose logarithm is uniform over [low, high]."""
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    kind = rng.choice(["step", "dense", "padded", "packed", "composite", "dropout", "dropout"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    form, coupled, reverse = rng.choice(["logit", "decay"]), rng.random() < 0.5, rng.random() < 0.3
    if kind == "dropout":
        rows, cols = spread(rng, 1, 40000), spread(rng, 1, 2000)
        return dict(op="dropout", rows=rows, cols=cols, dtype=dtype, p=round(rng.uniform(0.0, 0.9), 3), residual=rng.random() < 0.5)
    per_head = rng.choice([1, 1, 3, 16, 64, 128, 250])
    heads = max(1, spread(rng, 8, 2048) // per_head)
    if kind == "step":
        return dict(op="step", batch=spread(rng, 1, 768), channels=heads * per_head, heads=heads, dtype=dtype, form=form, coupled=coupled)
    more = dict(op="recurrence", dtype=dtype, form=form, coupled=coupled, reverse=reverse, train=rng.random() < 0.7, final_only=False)
    if kind == "composite":
        lists, mean = spread(rng, 100, 50000), rng.uniform(2, 40)
        channels = rng.choice([1, 2, 3, 4, 7, 16, 32])
        more.update(form="decay", coupled=True, reverse=True, final_only=True)
        return dict(more, layout="packed", batch=lists, rows=int(lists * mean) + 5, longest=512, channels=channels, heads=1)
    rows = spread(rng, 1, 20000)
    room = max(1, 60_000_000 // (rows * heads * per_head))     # under the largest listed case
    batch = spread(rng, 1, min(room, 64))
    if kind == "packed":
        return dict(more, layout="packed", batch=batch, rows=batch * rows + 3, longest=min(4 * rows + 1, batch * rows + 1),
                    channels=heads * per_head, heads=heads)
    return dict(more, layout=kind, batch=batch, rows=rows, longest=rows, channels=heads * per_head, heads=heads)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def total_rows(case):
    return case["rows"] if case["layout"] == "packed" else case["batch"] * case["rows"]


def sequence_lengths(case, seed):
    """Lengths of a padded or packed case's sequences (host): skewed, some empty, some of one row, some rows left over."""
    r = np.random.RandomState(seed % (1 << 31))
    n = case["batch"]
    if case["layout"] == "padded":
        lengths = r.randint(0, case["rows"] + 1, n)
        lengths[r.randint(n)] = case["rows"]
        return lengths.astype(np.int32)
    room = case["rows"] - min(3, case["rows"] - 1)
    weight = r.lognormal(0.0, 1.0, n) * (r.rand(n) > 0.03)
    lengths = np.minimum((weight / max(weight.sum(), 1e-9) * room).astype(np.int64), case["longest"])
    lengths[r.rand(n) < 0.02] = min(1, case["longest"])
    while lengths.sum() > room:
        lengths[lengths.argmax()] -= min(lengths.max(), lengths.sum() - room)
    return lengths.astype(np.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, dtype=dtype):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        state = dict(x=normal(*shape).requires_grad_(), grad=normal(*shape), p=case["p"],
                     rng=((seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), seed % 100000))
        if case["residual"]:
            state["residual"] = normal(*shape)
        return dict(state, case=case)

    def gates(*shape):
        if case["form"] == "logit":       # decays around 0.9, some short, some nearly 1
            return (torch.randn(shape, generator=g, device="cuda") * 1.5 + 2.3).to(dtype)
        if case["heads"] == 1:            # 1 - alpha of splats: most are faint, some nearly opaque
            return (1 - (torch.rand(shape, generator=g, device="cuda") ** 2 * 0.95 + 1 / 255)).to(dtype)
        return (1 - torch.rand(shape, generator=g, device="cuda") ** 2 * 0.5).to(dtype)

    b, d, heads = case["batch"], case["channels"], case["heads"]
    if case["op"] == "step":
        return dict(case=case, x=normal(b, d), gate=gates(b, heads), state=normal(b, d, dtype=torch.float32))
    lead = (case["rows"],) if case["layout"] == "packed" else (b, case["rows"])
    state = dict(case=case, x=normal(*lead, d), gate=gates(*lead, heads), state=normal(b, d, dtype=torch.float32))
    if case["layout"] != "dense":
        lengths = sequence_lengths(case, seed)
        if case["layout"] == "padded":
            state["lengths"] = torch.from_numpy(lengths).cuda()
        else:
            state["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).cuda()
    if case["train"]:
        for k in ("x", "gate", "state"):
            state[k].requires_grad_()
        state["grad_last"] = normal(b, d, dtype=torch.float32)
        if not case["final_only"]:
            state["grad_h"] = normal(*lead, d)
    return state


# ---- the operators ---------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "dropout":
        return run_dropout(state)
    if case["op"] == "step":
        return run_step(state)
    return run_recurrence(state)


def run_dropout(s):
    if own:
        import ds_splat_b200 as ds
        out = ds.dropout(s["x"], s["p"], s["rng"], residual=s.get("residual"))
        grad, = torch.autograd.grad(out, s["x"], s["grad"])
        return out.detach(), grad
    x, p = s["x"].detach(), s["p"]
    keep = philox_words(x.numel(), *s["rng"], x.device).view(x.shape) >= round(p * 2 ** 32)
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=torch.float32, device=x.device)
    out = torch.where(keep, x.float() * scale, 0.0)
    if "residual" in s:
        out = out + s["residual"].float()
    return out.to(x.dtype), torch.where(keep, s["grad"].float() * scale, 0.0).to(x.dtype)


def philox_words(count, seed, step, device):
    """Words 0 .. count - 1 of Philox4x32-10: block i // 4 has the counter (i // 4, step) and the key seed."""
    low = 0xFFFFFFFF
    quad = torch.arange((count + 3) // 4, device=device)
    c0, c1 = quad & low, quad >> 32
    c2, c3 = torch.full_like(quad, step & low), torch.full_like(quad, step >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low

    def product(m, c):      # both halves of a 32 x 32 bit product, without passing 63 bits
        return (m * (c >> 16) + (m * (c & 0xFFFF) >> 16)) >> 16, (m * (c & 0xFFFF) + ((m * (c >> 16) & 0xFFFF) << 16)) & low

    for _ in range(10):
        h0, l0 = product(0xD2511F53, c0)
        h1, l1 = product(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:count]


def decays(case, gate):
    """f and 1 - f in 32 bits, one value per channel."""
    gate = gate.float()
    f, k = (torch.sigmoid(gate), torch.sigmoid(-gate)) if case["form"] == "logit" else (gate, 1 - gate)
    per_head = case["channels"] // case["heads"]
    return f.repeat_interleave(per_head, -1), k.repeat_interleave(per_head, -1)


def run_step(s):
    case = s["case"]
    if own:
        import ds_splat_b200 as ds
        return ds.gated_recurrence_step(s["x"], s["gate"], s["state"], form=case["form"], coupled=case["coupled"]), s["state"]
    f, k = decays(case, s["gate"])
    x = s["x"].float()
    s["state"].copy_(f * s["state"] + (k * x if case["coupled"] else x))
    return s["state"].to(s["x"].dtype), s["state"]


def run_recurrence(s):
    case = s["case"]
    names = ("x", "gate", "state")
    if own:
        import ds_splat_b200 as ds
        h, last = ds.gated_recurrence(*(s[k] for k in names), offsets=s.get("offsets"), lengths=s.get("lengths"), form=case["form"],
                                      coupled=case["coupled"], reverse=case["reverse"], final_only=case["final_only"])
        out = dict(last=last.detach()) if case["final_only"] else dict(h=h.detach(), last=last.detach())
        if case["train"]:
            outs, grads = ((last,), (s["grad_last"],)) if case["final_only"] else ((h, last), (s["grad_h"], s["grad_last"]))
            out.update(zip(("dx", "dgate", "dstate"), torch.autograd.grad(outs, [s[k] for k in names], grads)))
        return out

    # rows in the order of the recurrence, all sequences one behind the other
    flip = (lambda t: t.flip(0)) if case["reverse"] else (lambda t: t)
    n, d, heads = total_rows(case), case["channels"], case["heads"]
    x, gate = (flip(s[k].detach().reshape(n, -1)) for k in ("x", "gate"))
    state = flip(s["state"].detach())
    first, end, owner, inside = row_tables(s, n, x.device)
    f, k = decays(case, gate)
    xf = x.float()
    i = k * xf if case["coupled"] else xf
    start = torch.where(first[:, None], state[owner], 0.0)              # the state that reaches a sequence's first row
    open_f = torch.where(first[:, None] | ~inside[:, None], 0.0, f)
    h = scan(open_f, torch.where(inside[:, None], i + torch.where(first[:, None], f * start, 0.0), 0.0), case["longest"])
    last = state.clone()
    last[owner[end]] = h[end]
    put = lambda t, like: flip(torch.where(inside[:, None], t, 0.0)).to(like.dtype).view(like.shape)  # noqa: E731
    out = dict(last=flip(last)) if case["final_only"] else dict(h=put(h, s["x"]), last=flip(last))
    if not case["train"]:
        return out

    before = torch.where(first[:, None], start, torch.cat([h[:1], h[:-1]]))          # h_{t-1}
    grad_last = flip(s["grad_last"])
    g = torch.zeros_like(h) if case["final_only"] else flip(s["grad_h"].reshape(n, -1)).float()
    g = torch.where(inside[:, None], g + torch.where(end[:, None], grad_last[owner], 0.0), 0.0)
    f_next = torch.cat([f[1:], f[:1]])
    f_next = torch.where(end[:, None] | ~inside[:, None], 0.0, f_next)
    g = scan(f_next.flip(0), g.flip(0), case["longest"]).flip(0)
    df = (g * (before - xf if case["coupled"] else before))
    if case["form"] == "logit":
        df = df * f * k
    dstate = grad_last.clone()
    dstate[owner[first]] = (f * g)[first]
    out.update(dx=put(k * g if case["coupled"] else g, s["x"]), dgate=put(df.view(n, heads, d // heads).sum(-1), s["gate"]),
               dstate=flip(dstate))
    return out


def row_tables(s, n, device):
    """Per row, in the order of the recurrence: whether it is its sequence's first, its last, which sequence it belongs to, and
    whether it belongs to any."""
    case = s["case"]
    row = torch.arange(n, device=device)
    if "offsets" in s:
        offsets = s["offsets"].long()
        starts, ends = offsets[:-1], offsets[1:]
    else:
        starts = torch.arange(case["batch"], device=device) * case["rows"]
        ends = starts + (s["lengths"].long() if "lengths" in s else case["rows"])
    if case["reverse"]:
        starts, ends = (n - ends).flip(0), (n - starts).flip(0)
    owner = (torch.searchsorted(ends, row, right=True)).clamp_(max=case["batch"] - 1)
    inside = (row >= starts[owner]) & (row < ends[owner])
    return inside & (row == starts[owner]), inside & (row == ends[owner] - 1), owner, inside


def scan(f, b, longest):
    """h_t = f_t h_{t-1} + b_t over dimension 0 by doubling the span that each row has summed up."""
    span = 1
    while span < longest and span < f.shape[0]:
        b = torch.cat([b[:span], b[span:] + f[span:] * b[:-span]])
        f = torch.cat([f[:span], f[span:] * f[:-span]])
        span *= 2
    return b


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]                        # x, its gradient's source, both results (and the residual)
        return dict(bytes=(5 if case["residual"] else 4) * n * e, flops=4 * n)
    if case["op"] == "step":
        n = case["batch"] * case["channels"]
        return dict(bytes=n * (2 * e + 8) + case["batch"] * case["heads"] * e, flops=4 * n)
    n, d, heads = total_rows(case), case["channels"], case["heads"]
    states = case["batch"] * d * 4
    h = 0 if case["final_only"] else n * d
    if not case["train"]:
        return dict(bytes=(n * (d + heads) + h) * e + 2 * states, flops=4 * n * d)
    return dict(bytes=(2 * n * (d + heads) + 2 * h) * e + 4 * states, flops=16 * n * d)


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        keep = torch.from_numpy(exact_words(case["rows"] * case["cols"], *s["rng"]) >= round(case["p"] * 2 ** 32)).cuda()
        keep = keep.view(case["rows"], case["cols"]).double()
        q = 1.0 - case["p"]
        out = keep * s["x"].detach().double() / q + (s["residual"].double() if case["residual"] else 0.0)
        return out, keep * s["grad"].double() / q
    d, per_head = case["channels"], case["channels"] // case["heads"]
    wide = lambda t: torch.repeat_interleave(t.detach().double(), per_head, -1)  # noqa: E731
    if case["op"] == "step":
        f = wide(s["gate"])
        f = 1 / (1 + torch.exp(-f)) if case["form"] == "logit" else f
        h = f * s["state"].double() + (1 - f if case["coupled"] else 1) * s["x"].double()
        return h, h

    # one sequence after the other in time, all sequences side by side: [time, sequence, channel]
    n, b = total_rows(case), case["batch"]
    if case["layout"] == "packed":
        o = s["offsets"].cpu().numpy().astype(np.int64)
        begin, count = o[:-1], np.diff(o)
    else:
        begin = np.arange(b, dtype=np.int64) * case["rows"]
        count = s["lengths"].cpu().numpy().astype(np.int64) if case["layout"] == "padded" else np.full(b, case["rows"], np.int64)
    span = int(count.max())
    if span * b * d > 700_000_000 or span > 200_000:
        return None
    t = np.arange(span)[:, None]
    row = begin + (count - 1 - t if case["reverse"] else t)
    there = torch.from_numpy(t < count).cuda()
    row = torch.from_numpy(np.where(t < count, row, 0)).cuda()
    there3 = there[:, :, None]
    at = lambda v: v.detach().reshape(n, -1).double()[row]  # noqa: E731
    gate, x = at(s["gate"]), at(s["x"])
    f = 1 / (1 + torch.exp(-gate)) if case["form"] == "logit" else gate
    slope = torch.repeat_interleave(f * (1 - f) if case["form"] == "logit" else torch.ones_like(f), per_head, -1)
    del gate
    f = torch.repeat_interleave(f, per_head, -1)
    h0 = s["state"].detach().double()
    hs = torch.empty(span + 1, b, d, dtype=torch.float64, device="cuda")
    hs[0] = h0
    i = torch.where(there3, (1 - f) * x if case["coupled"] else x, 0.0)
    stay = torch.where(there3, f, 1.0)                          # a sequence that has ended keeps its state
    for a, fa, ia, to in zip(hs[:-1].unbind(0), stay.unbind(0), i.unbind(0), hs[1:].unbind(0)):
        torch.addcmul(ia, fa, a, out=to)
    del i

    def back(v, like):                                          # [time, sequence, ...] to the rows it came from
        flat = torch.zeros(n, v.shape[-1], dtype=torch.float64, device="cuda")
        flat[row[there]] = v[there]
        return flat.view(like.shape)

    out = dict(last=hs[-1].clone()) if case["final_only"] else dict(h=back(hs[1:], s["x"]), last=hs[-1].clone())
    if not case["train"]:
        return out
    dh = torch.zeros_like(stay) if case["final_only"] else torch.where(there3, at(s["grad_h"]), 0.0)
    gs = dh                                                     # becomes g_t, in place
    q = s["grad_last"].double()
    for ga, fa in zip(reversed(gs.unbind(0)), reversed(stay.unbind(0))):
        ga.add_(q)
        q = fa * ga
    out["dx"] = back((1 - f) * gs if case["coupled"] else gs, s["x"])
    df = gs * (hs[:-1] - x if case["coupled"] else hs[:-1]) * slope
    out["dgate"] = back(df.view(span, b, case["heads"], per_head).sum(-1), s["gate"])
    out["dstate"] = q
    return out


def exact_words(count, seed, step):
    """Philox4x32-10 again, in unsigned 64-bit arithmetic on the host."""
    u = np.uint64
    low, half = u(0xFFFFFFFF), u(32)
    quad = np.arange(-(-count // 4), dtype=u)
    a, b = quad & low, quad >> half
    c, d = np.full_like(quad, u(step % 2 ** 32)), np.full_like(quad, u(step // 2 ** 32 % 2 ** 32))
    key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
    for turn in range(10):
        p, r = a * u(0xD2511F53), c * u(0xCD9E8D57)
        a, b, c, d = (r >> half) ^ b ^ u(key[0]), r & low, (p >> half) ^ d ^ u(key[1]), p & low
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack([a, b, c, d], 1).reshape(-1)[:count]
