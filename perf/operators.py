"""The operators beside tb.matmul that a mixture of experts and a block-scaled
8-bit layer call, as measured cases: their plain forms in torch, the calls a
user's program makes, and their values in 64 bits.

  grouped_matmul        C[rows of e] = A[rows of e] · B[e]          (f16 / bf16)
  grouped_matmul_wgrad  G[e] = A[rows of e]^T · D[rows of e]        (f16 / bf16)
  quantize_fp8          S = m / 448, Q = e4m3(448 X / m), m = max(max|block|, 448 · 2^-63)
  matmul_fp8            C = Σ_b SA[·, b] SB[b, ·] (A_b · B_b), b = blocks of 128 along K
  grouped_matmul_fp8    the same for the rows of each expert

The rows of expert e are [offsets[e], offsets[e + 1]) of T rows; the offsets
live on the GPU, as a router leaves them. Rows outside every expert (before
offsets[0], behind offsets[E]) keep what C held.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_FP8 = torch.float8_e4m3fn
_MAX = 448.0           # largest e4m3 value
_LEAST = 2.0 ** -63    # least scale: the product of two scales stays a normal f32


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one decoding step of a small batch: eight rows over the experts, each weight read once
        dict(name="grouped decode 8 rows", op="grouped", t=8, spare=0, e=8, k=1024, n=1024, dtype="bf16", out="bf16",
             weights="kn"),
        # a decoding step of a larger batch over many experts with weights kept as n × k
        dict(name="grouped decode 96 rows", op="grouped", t=96, spare=0, e=32, k=2048, n=1408, dtype="f16",
             out="f16", weights="nk"),
        # a ragged prompt chunk, odd widths, some rows padded behind the last expert
        dict(name="grouped prompt odd", op="grouped", t=4099, spare=61, e=16, k=1032, n=1288, dtype="f16", out="f32",
             weights="kn"),
        # a training batch through the experts' first product
        dict(name="grouped training", op="grouped", t=16384, spare=0, e=8, k=4096, n=4096, dtype="bf16", out="bf16",
             weights="kn"),
        # the experts' weight gradients of a short, odd batch
        dict(name="wgrad short", op="wgrad", t=777, spare=0, e=8, k=512, n=768, dtype="bf16", out="f32"),
        # the experts' weight gradients of a training batch
        dict(name="wgrad training", op="wgrad", t=16384, spare=0, e=8, k=4096, n=2048, dtype="bf16", out="bf16"),
        # activations of one decoding step
        dict(name="quantize 16 rows", op="quantize", r=16, c=4096, dtype="bf16", block="row"),
        # activations of a training batch, blocks along the rows' axis as a weight gradient reads them
        dict(name="quantize training", op="quantize", r=16384, c=8192, dtype="bf16", block="column"),
        # a decoding step through one 8-bit layer
        dict(name="fp8 decode 16 rows", op="fp8", m=16, n=4096, k=4096, out="bf16", form="forward"),
        # the headline size of the matmul family in 8 bits
        dict(name="fp8 8192", op="fp8", m=8192, n=8192, k=8192, out="bf16", form="forward"),
        # a decoding step of 8-bit experts
        dict(name="grouped fp8 decode", op="grouped_fp8", t=64, spare=0, e=16, k=2048, n=2048, out="bf16",
             weights="nk"),
        # a prompt through 8-bit experts
        dict(name="grouped fp8 prompt", op="grouped_fp8", t=8200, spare=56, e=16, k=4096, n=2048, out="bf16",
             weights="nk"),
    ]


def _spread(rng, lo, hi):
    """A whole number, evenly spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi, unit):
    """A row length: mostly whole units of 16 bytes, one in five any number."""
    v = _spread(rng, lo, hi)
    return v if rng.random() < 0.2 else max(unit, v // unit * unit)


def draw(rng):
    op = rng.choice(["grouped", "grouped", "wgrad", "quantize", "fp8", "grouped_fp8"])
    if op == "quantize":
        return dict(op=op, r=_spread(rng, 1, 16384), c=_width(rng, 128, 8192, 8),
                    dtype=rng.choice(["bf16", "f16", "f32"]), block=rng.choice(["row", "column", "square"]))
    if op == "fp8":
        form = rng.choice(["forward", "forward", "input gradient", "weight gradient"])
        return dict(op=op, m=_spread(rng, 1, 8192), n=_width(rng, 128, 8192, 16), k=_width(rng, 128, 8192, 16),
                    out=rng.choice(["bf16", "f16", "f32"]), form=form)
    unit = 16 if op == "grouped_fp8" else 8
    t = _spread(rng, 1, 16384)
    case = dict(op=op, t=t, spare=rng.choice([0, 0, 1 + t // 50]), e=_spread(rng, 1, 64),
                k=_width(rng, 128, 4096, unit), n=_width(rng, 128, 4096, unit),
                out=rng.choice(["bf16", "f16", "f32"]))
    if op != "grouped_fp8":
        case["dtype"] = rng.choice(["bf16", "f16"])
        if case["out"] != "f32":
            case["out"] = case["dtype"]
    if op != "wgrad":
        case["weights"] = rng.choice(["kn", "nk"])
    while case["e"] * case["k"] * case["n"] > 8 * 4096 * 4096:
        case["e"] = (case["e"] + 1) // 2
    return case


def _sizes(case, seed):
    """Rows of each expert: uneven, one expert of four or more without any."""
    t, e = case["t"], case["e"]
    r = np.random.RandomState(seed % (1 << 31))
    idle = int(r.randint(e)) if e >= 4 else -1
    busy = np.array([i for i in range(e) if i != idle])
    sizes = np.zeros(e, dtype=np.int64)
    if t <= len(busy):
        sizes[r.permutation(busy)[:t]] = 1
        return sizes
    sizes[busy] = 1
    p = np.exp(0.25 * r.standard_normal(len(busy)))
    sizes[busy] += r.multinomial(t - len(busy), p / p.sum())
    return sizes


def _busy(case):
    return min(case["t"], case["e"] - 1 if case["e"] >= 4 else case["e"])


# ----------------------------------------------------------------- the inputs

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g, rows, cols):
    """Normal values whose size differs from column to column, as a layer's inputs do."""
    x = _randn(g, rows, cols)
    x *= torch.exp(0.5 * _randn(g, 1, cols))
    return x


def _quantized(x, br, bc):
    """Q and S of x (…, R, C) in blocks of br × bc, by the formula."""
    q, s = _quantize(x, br, bc)
    return q.to(_FP8), s


def _padded(q):
    """The same 8-bit matrix with rows that begin on 16-byte boundaries, as a program that makes its own buffers has it."""
    cols = q.shape[-1]
    wide = torch.zeros(*q.shape[:-1], (cols + 15) // 16 * 16, device=q.device, dtype=torch.uint8).view(_FP8)
    wide.view(torch.uint8)[..., :cols] = q.view(torch.uint8)
    return wide[..., :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op = case["op"]
    if op == "quantize":
        r, c = case["r"], case["c"]
        br, bc = _blocks(case)
        return dict(case=case, x=_activations(g, r, c).to(_TYPES[case["dtype"]]),
                    q=torch.zeros(r, c, device="cuda", dtype=torch.uint8).view(_FP8),
                    s=torch.zeros(-(-r // br), -(-c // bc), device="cuda"))
    if op == "fp8":
        m, n, k, form = case["m"], case["n"], case["k"], case["form"]
        c = torch.zeros(m, n, device="cuda", dtype=_TYPES[case["out"]])
        if form == "weight gradient":  # the batch runs along k: both sides in blocks of 128 rows of the batch
            a, sa = _quantized(_activations(g, k, m), 128, 1)
            b, sb = _quantized(_activations(g, k, n), 128, 1)
            return dict(case=case, a=_padded(a).t(), sa=sa.t(), b=_padded(b), sb=sb, c=c)
        a, sa = _quantized(_activations(g, m, k), 1, 128)
        if form == "forward":          # weights kept as n × k
            b, sb = _quantized(_randn(g, n, k) / math.sqrt(k), 128, 128)
            return dict(case=case, a=_padded(a), sa=sa, b=_padded(b).t(), sb=sb.t(), c=c)
        b, sb = _quantized(_randn(g, k, n) / math.sqrt(k), 128, 128)  # the same weights read along their rows
        return dict(case=case, a=_padded(a), sa=sa, b=_padded(b), sb=sb, c=c)
    t, e, k, n = case["t"], case["e"], case["k"], case["n"]
    sizes = _sizes(case, seed)
    ends = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    state = dict(case=case, offsets=torch.from_numpy(ends).cuda(), most=int(sizes.max()))
    rows = t + case["spare"]
    if op == "grouped_fp8":
        a, sa = _quantized(_activations(g, rows, k), 1, 128)
        nk = case["weights"] == "nk"
        w, sw = _quantized(_randn(g, e, *((n, k) if nk else (k, n))) / math.sqrt(k), 128, 128)
        w = _padded(w)
        state.update(a=_padded(a), sa=sa, b=w.transpose(1, 2) if nk else w, sb=sw.transpose(1, 2) if nk else sw,
                     c=_randn(g, rows, n).to(_TYPES[case["out"]]))
        return state
    dt = _TYPES[case["dtype"]]
    state["a"] = _activations(g, rows, k).to(dt)
    if op == "wgrad":
        state["d"] = (_randn(g, rows, n) / math.sqrt(t)).to(dt)
        state["g"] = torch.zeros(e, k, n, device="cuda", dtype=_TYPES[case["out"]])
        return state
    if case["weights"] == "nk":
        state["b"] = (_randn(g, e, n, k) / math.sqrt(k)).to(dt).transpose(1, 2)
    else:
        state["b"] = (_randn(g, e, k, n) / math.sqrt(k)).to(dt)
    state["c"] = _randn(g, rows, n).to(_TYPES[case["out"]])
    return state


# ---------------------------------------------------------------- plain forms

def _blocks(case):
    return {"row": (1, 128), "column": (128, 1), "square": (128, 128)}[case["block"]]


def _quantize(x, br, bc):
    """(448 X / m in f32, to be rounded to e4m3, and S in f32). 448 X is taken as 0.4375 X, against m / 1024: exact for
    16-bit X and never infinite, so that a quotient on the border between two e4m3 values comes out on it."""
    *lead, r, c = x.shape
    rb, cb = -(-r // br), -(-c // bc)
    p = torch.nn.functional.pad(x.float(), (0, cb * bc - c, 0, rb * br - r))
    p = p.view(*lead, rb, br, cb, bc)
    most = p.abs().amax(dim=(-3, -1)).clamp(min=_MAX * _LEAST)
    s = most / torch.full_like(most, _MAX)  # a tensor divisor: torch multiplies by 1 / number
    q = (p * (_MAX / 1024)) / (most / 1024)[..., :, None, :, None]
    return q.view(*lead, rb * br, cb * bc)[..., :r, :c], s


def _values(q, s):
    """Q · S in f32, each scale spread over its block (the block's extent shows in the shapes)."""
    r, c = q.shape[-2:]
    v = q.float()
    rows = torch.arange(r, device=q.device) // (1 if s.shape[-2] == r else 128)
    cols = torch.arange(c, device=q.device) // (1 if s.shape[-1] == c else 128)
    return v * s[..., rows, :][..., cols]


def _owner(offsets, rows):
    """Per row: its expert, its place among the expert's rows, and whether it has one."""
    t = torch.arange(rows, device=offsets.device)
    e = torch.searchsorted(offsets, t, right=True) - 1
    has = (e >= 0) & (e < offsets.numel() - 1)
    e = e.clamp(0, offsets.numel() - 2)
    return e, t - offsets[e], has


def _by_expert(x, offsets, most):
    """x's rows as (experts, most, columns), zeros behind each expert's last row."""
    place = torch.arange(most, device=x.device)
    rows = offsets[:-1, None] + place
    held = rows < offsets[1:, None]
    return torch.where(held[..., None], x[rows.clamp(max=x.shape[0] - 1)], torch.zeros((), device=x.device))


def _plain_grouped(a, b, c, offsets, most):
    e, place, has = _owner(offsets, a.shape[0])
    y = torch.bmm(_by_expert(a, offsets, most), b)
    c.copy_(torch.where(has[:, None], y[e, place.clamp(0, most - 1)], c.float()))
    return c


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    if op == "grouped":
        return _plain_grouped(state["a"].float(), state["b"].float(), state["c"], state["offsets"], state["most"])
    if op == "wgrad":
        a = _by_expert(state["a"].float(), state["offsets"], state["most"])
        d = _by_expert(state["d"].float(), state["offsets"], state["most"])
        state["g"].copy_(torch.bmm(a.transpose(1, 2), d))
        return state["g"]
    if op == "quantize":
        q, s = _quantize(state["x"], *_blocks(state["case"]))
        return {"q": q.to(_FP8), "s": s}
    if op == "fp8":
        state["c"].copy_(_values(state["a"], state["sa"]) @ _values(state["b"], state["sb"]))
        return state["c"]
    return _plain_grouped(_values(state["a"], state["sa"]), _values(state["b"], state["sb"]), state["c"],
                          state["offsets"], state["most"])


# ------------------------------------------------------------ the user's calls

def _own(op, s):
    import mini_triton_nvgpu_v1_b200 as tb
    if op == "grouped":
        return tb.grouped_matmul(s["a"], s["b"], s["c"], s["offsets"], beta=0)
    if op == "wgrad":
        return tb.grouped_matmul_wgrad(s["a"], s["d"], s["g"], s["offsets"], beta=0)
    if op == "quantize":
        tb.quantize_fp8(s["x"], s["q"], s["s"], block=_blocks(s["case"]))
        return {"q": s["q"], "s": s["s"]}
    if op == "fp8":
        return tb.matmul_fp8(s["a"], s["sa"], s["b"], s["sb"], s["c"], beta=0)
    return tb.grouped_matmul_fp8(s["a"], s["sa"], s["b"], s["sb"], s["c"], s["offsets"], beta=0)


# ---------------------------------------------------------- floors and values

def work(case):
    """Bytes read and written once, and multiply-adds counted as two operations."""
    op = case["op"]
    size = {"f16": 2, "bf16": 2, "f32": 4}
    if op == "quantize":
        br, bc = _blocks(case)
        r, c = case["r"], case["c"]
        return {"bytes": r * c * (size[case["dtype"]] + 1) + 4 * -(-r // br) * -(-c // bc), "flops": 2 * r * c}
    if op == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // 128)
        scales = kb * (m + n) if case["form"] == "weight gradient" else kb * (m + -(-n // 128))
        return {"bytes": m * k + k * n + m * n * size[case["out"]] + 4 * scales, "flops": 2 * m * n * k}
    t, e, k, n = case["t"], case["e"], case["k"], case["n"]
    if op == "wgrad":
        return {"bytes": 2 * t * (k + n) + e * k * n * size[case["out"]], "flops": 2 * t * k * n}
    width = 1 if op == "grouped_fp8" else 2
    scales = 4 * -(-k // 128) * (t + _busy(case) * -(-n // 128)) if op == "grouped_fp8" else 0
    return {"bytes": width * (t * k + _busy(case) * k * n) + t * n * size[case["out"]] + scales,
            "flops": 2 * t * k * n}


def _e4m3_64(v):
    """The nearest e4m3 value (ties to even) of each f64 value in [-448, 448]."""
    m, x = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(x - 4, min=-9))
    return torch.round(v / step) * step


def _spread64(q, s, br, bc):
    v = q.double()
    for axis, b in ((-2, br), (-1, bc)):
        s = s.double().repeat_interleave(b, dim=axis).narrow(axis, 0, q.shape[axis])
    return v * s


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = s["x"].double()
        r, c = x.shape
        br, bc = _blocks(case)
        b = x.new_zeros(-(-r // br) * br, -(-c // bc) * bc)
        b[:r, :c] = x
        most = b.abs().reshape(b.shape[0] // br, br, -1, bc).permute(0, 2, 1, 3).flatten(2).max(dim=2).values
        most = torch.clamp(most, min=_MAX * _LEAST)
        over = most.repeat_interleave(br, 0)[:r].repeat_interleave(bc, 1)[:, :c]
        return {"q": _e4m3_64(x * _MAX / over), "s": most / _MAX}
    if op == "fp8":
        gradient = case["form"] == "weight gradient"
        a = _spread64(s["a"], s["sa"], 1, 128)
        b = _spread64(s["b"], s["sb"], 128, 1 if gradient else 128)
        return a @ b
    ends = s["offsets"].tolist()
    if op == "wgrad":
        return torch.stack([s["a"][lo:hi].double().t() @ s["d"][lo:hi].double() for lo, hi in zip(ends, ends[1:])])
    c = s["c"].double()
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if op == "grouped_fp8":
            c[lo:hi] = _spread64(s["a"][lo:hi], s["sa"][lo:hi], 1, 128) @ _spread64(s["b"][e], s["sb"][e], 128, 128)
        else:
            c[lo:hi] = s["a"][lo:hi].double() @ s["b"][e].double()
    return c
