"""GPU: 8-bit operands with a scale per block of 128: the quantiser and the
dense and grouped products, against the formulas in 64 bits.

Where the e4m3 values are small whole numbers and the scales powers of two,
every product and partial sum is exact in f32: the f32 output has to be equal,
a 16-bit output the exact value rounded once."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

OUT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def _type(name):
    import torch
    return getattr(torch, OUT[name])


def _gen(seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _blocks(n):
    return -(-n // 128)


# ------------------------------------------------------------------ quantiser

def _quantized64(x, br, bc):
    """(Q, S) from the definition in 64 bits; x [rows, cols] without NaN or infinities."""
    import torch
    r, c = x.shape
    p = torch.zeros(_blocks(r) * 128, _blocks(c) * 128, device=x.device, dtype=torch.float64)
    p[:r, :c] = x.double().abs()
    rb, cb = -(-r // br), -(-c // bc)
    p = p[:rb * br, :cb * bc] if br == 128 or bc == 128 else p
    m = p[:rb * br, :cb * bc].reshape(rb, br, cb, bc).amax(dim=(1, 3)).clamp(min=448 * 2.0 ** -63)
    over = m.repeat_interleave(br, 0)[:r].repeat_interleave(bc, 1)[:, :c]
    v = x.double() * 448 / over
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 4, min=-9))  # e4m3: 4 significant bits, least step 2^-9
    return torch.round(v / step) * step, m / 448


@pytest.mark.parametrize("block", [(1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r,c", [(1, 1), (1, 128), (3, 7), (16, 4096), (127, 129), (128, 128), (129, 131), (500, 1000),
                                 (1025, 264)])
def test_quantize(cuda, block, dtype, r, c):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = _gen(r * 31 + c)
    x = torch.randn(r, c, generator=g, device="cuda") * torch.exp(2 * torch.randn(1, c, generator=g, device="cuda"))
    x = x.to(_type(dtype))
    Q, S = tb.quantize_fp8(x, block=block)
    q, s = _quantized64(x, *block)
    assert Q.dtype == torch.float8_e4m3fn and Q.stride(0) % 16 == 0 or r == 1
    # S = m / 448 rounded once to f32
    assert torch.equal(S, s.float())
    if dtype == "f32":
        # 0.4375·X and the quotient are each rounded to f32 (2^-24): a quotient that near to the border of two
        # e4m3 values may go to either
        v = Q.double()
        near = (v - q).abs() / q.abs().clamp(min=2.0 ** -6) <= 2.0 ** -3
        assert near.all() and (v != q).double().mean() <= 1e-4
    else:
        assert torch.equal(Q.double(), q)


def test_quantize_ties_and_extremes(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    # a block whose maximum is 448: Q is X rounded to e4m3, with every tie between neighbours
    grid = torch.arange(0, 127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    x = torch.cat([grid, (grid[1:] + grid[:-1]) / 2])
    x = torch.cat([x, -x, x.new_zeros(-2 * len(x) % 127)]).reshape(-1, 127)
    x = torch.cat([x, torch.full_like(x[:, :1], 448)], dim=1).float()
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        y = x.to(dt)
        Q, S = tb.quantize_fp8(y)
        q, s = _quantized64(y, 1, 128)
        assert torch.equal(Q.double(), q) and torch.equal(S, torch.ones_like(S))
    # zeros, the least and the greatest values of each type
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        i = torch.finfo(dt)
        rows = torch.tensor([[0.0, 0.0], [i.max, -i.max], [i.max, i.tiny], [i.tiny, 0.0], [i.max, 1.0]],
                            device="cuda", dtype=torch.float64)
        y = rows.repeat(1, 64).to(dt)
        Q, S = tb.quantize_fp8(y)
        q, s = _quantized64(y, 1, 128)
        assert torch.equal(Q.double(), q) and torch.equal(S, s.float()), dt
    Q, S = tb.quantize_fp8(torch.zeros(200, 300, device="cuda"), block=(128, 128))
    assert not Q.float().any() and (S == 2.0 ** -63).all()


@pytest.mark.parametrize("block", [(1, 128), (128, 1), (128, 128)])
def test_quantize_nan_and_infinity(cuda, block):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    x = torch.randn(256, 256, generator=_gen(1), device="cuda").bfloat16()
    clean_q, clean_s = tb.quantize_fp8(x, block=block)
    x[5, 7] = float("nan")
    x[200, 130] = float("-inf")
    Q, S = tb.quantize_fp8(x, block=block)
    br, bc = block
    nan, inf = torch.zeros(256, 256, dtype=torch.bool, device="cuda"), torch.zeros(256, 256, dtype=torch.bool, device="cuda")
    nan[5 // br * br:5 // br * br + br, 7 // bc * bc:7 // bc * bc + bc] = True
    inf[200 // br * br:200 // br * br + br, 130 // bc * bc:130 // bc * bc + bc] = True
    v = Q.float()
    assert torch.isnan(v[nan]).all() and torch.isnan(S[5 // br, 7 // bc])
    assert torch.isinf(S[200 // br, 130 // bc]) and torch.isnan(v[200, 130])
    inf[200, 130] = False
    assert not v[inf].any()
    inf[200, 130] = True
    assert torch.equal(v[~nan & ~inf], clean_q.float()[~nan & ~inf])


def test_quantize_strides_and_batches(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = _gen(2)
    for rows, cols, skip in ((130, 264, 0), (130, 264, 8), (130, 264, 1), (77, 45, 3)):
        for block in ((1, 128), (128, 1), (128, 128)):
            whole = torch.randn(3, rows + 1, cols + skip, generator=g, device="cuda").half()
            x = whole[:, :rows, skip:]
            q = torch.zeros(3, rows, cols + 2 * skip, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
            s = torch.zeros(3, -(-cols // block[1]), -(-rows // block[0]), device="cuda").transpose(1, 2)
            Q, S = tb.quantize_fp8(x, q[:, :, skip:skip + cols], s, block=block)
            for b in range(3):
                eq, es = _quantized64(x[b], *block)
                assert torch.equal(Q[b].double(), eq) and torch.equal(S[b], es.float())
            around = q.view(torch.uint8).clone()
            around[:, :, skip:skip + cols] = 0
            assert not around.any()
    for shape in ((0, 128), (4, 0), (0, 4, 128)):
        tb.quantize_fp8(torch.zeros(*shape, device="cuda"))


# ------------------------------------------------------------------- products

def _e4m3(shape, g, most=3):
    import torch
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").float().to(torch.float8_e4m3fn)


def _powers(shape, g):
    import torch
    return torch.exp2(torch.randint(-2, 3, shape, generator=g, device="cuda").float())


def _wide(q):
    """The same values in rows that begin on 16-byte boundaries."""
    import torch
    w = torch.zeros(*q.shape[:-1], (q.shape[-1] + 15) // 16 * 16, device="cuda", dtype=torch.uint8)
    w[..., :q.shape[-1]] = q.view(torch.uint8)
    return w.view(torch.float8_e4m3fn)[..., :q.shape[-1]]


def _spread(q, s, rows_per, cols_per):
    r, c = q.shape[-2:]
    s = s.double().repeat_interleave(rows_per, -2)[..., :r, :].repeat_interleave(cols_per, -1)[..., :c]
    return q.double() * s


def _dense(g, m, n, k, a_col, b_col, a_per, b_per, wide=True, real=False):
    import torch
    lay = _wide if wide else (lambda q: q)
    if real:
        mk = lambda sh: torch.randn(sh, generator=g, device="cuda").mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn)
        sc = lambda sh: torch.exp(torch.randn(sh, generator=g, device="cuda"))
    else:
        mk, sc = (lambda sh: _e4m3(sh, g)), (lambda sh: _powers(sh, g))
    A = lay(mk((k, m))).t() if a_col else lay(mk((m, k)))
    B = lay(mk((n, k))).t() if b_col else lay(mk((k, n)))
    SA = sc((-(-m // a_per), _blocks(k)))
    SB = sc((_blocks(k), -(-n // b_per)))
    return A, SA, B, SB


SIZES = [(1, 1, 1), (1, 512, 1024), (5, 96, 136), (16, 4096, 512), (33, 200, 129), (96, 1000, 260), (128, 128, 128),
         (130, 257, 1000), (700, 2568, 200), (2000, 2600, 390)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("a_col,b_col,a_per,b_per", [(0, 1, 1, 128), (0, 0, 1, 128), (1, 0, 1, 1), (0, 1, 128, 128),
                                                     (1, 1, 128, 1), (0, 1, 1, 1)])
def test_matmul_fp8(cuda, m, n, k, a_col, b_col, a_per, b_per):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = _gen(m + n + k)
    A, SA, B, SB = _dense(g, m, n, k, a_col, b_col, a_per, b_per)
    ref = _spread(A, SA, a_per, 128) @ _spread(B, SB, 128, b_per)
    for out, beta in (("f32", 1), ("bf16", 0), ("f16", 1)):
        C = torch.randint(-9, 10, (m, n), generator=g, device="cuda").to(_type(out))
        want = (ref + beta * C.double()).to(C.dtype)
        got = tb.matmul_fp8(A, SA, B, SB, C, beta=beta)
        tb.device_status()
        assert got is C and torch.equal(C, want)


@pytest.mark.parametrize("m,n,k", [(7, 200, 700), (140, 520, 650), (1500, 2600, 1100)])
@pytest.mark.parametrize("a_col,b_col,a_per,b_per", [(0, 1, 1, 128), (1, 0, 1, 1)])
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
def test_matmul_fp8_real_values(cuda, m, n, k, a_col, b_col, a_per, b_per, out):
    """128 additions inside a block and one per block, each off by at most one unit in the last place of f32 (2^-23),
    the two scales' product and its product with the block's sum (2^-23 each); then half a step of the output."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    A, SA, B, SB = _dense(_gen(m), m, n, k, a_col, b_col, a_per, b_per, real=True)
    SA, SB = SA * 1e-3, SB * 1e-3
    a, b = _spread(A, SA, a_per, 128), _spread(B, SB, 128, b_per)
    ref, most = a @ b, a.abs() @ b.abs()
    C = torch.zeros(m, n, device="cuda", dtype=_type(out))
    tb.matmul_fp8(A, SA, B, SB, C, beta=0)
    sums = (128 + _blocks(k) + 3) * 2.0 ** -23 * most
    tol = sums + torch.finfo(C.dtype).eps / 2 * (ref.abs() + sums) + 2.0 ** -25
    assert ((C.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("sizes,k,n", [([1], 128, 64), ([0, 3, 0, 5], 200, 136), ([1, 2, 0, 1, 7, 1], 2048, 512),
                                       ([33, 128, 96, 140], 392, 1000), ([300, 0, 257, 700, 256, 487], 264, 2568),
                                       ([i % 4 for i in range(200)], 130, 130)])
@pytest.mark.parametrize("nk,b_per", [(1, 128), (0, 128), (1, 1)])
def test_grouped_matmul_fp8(cuda, sizes, k, n, nk, b_per):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = _gen(k + n)
    ends = [3]
    for s in sizes:
        ends.append(ends[-1] + s)
    rows, E = ends[-1] + 4, len(sizes)
    off = torch.tensor(ends, dtype=torch.int32, device="cuda")
    A, SA = _wide(_e4m3((rows, k), g)), _powers((rows, _blocks(k)), g)
    A.view(torch.uint8)[ends[-1]:] = 0x7f  # NaN
    SA[:3] = float("nan")
    B = _wide(_e4m3((E, n, k), g)).transpose(1, 2) if nk else _wide(_e4m3((E, k, n), g))
    SB = _powers((E, _blocks(k), -(-n // b_per)), g)
    for out, beta in (("f32", 1), ("bf16", 0)):
        C = torch.randint(-9, 10, (rows, n), generator=g, device="cuda").to(_type(out))
        want = C.double()
        for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
            want[lo:hi] = (_spread(A[lo:hi], SA[lo:hi], 1, 128) @ _spread(B[e], SB[e], 128, b_per)
                           + beta * C[lo:hi].double())
        tb.grouped_matmul_fp8(A, SA, B, SB, C, off, beta=beta)
        tb.device_status()
        assert torch.equal(C, want.to(C.dtype))


def test_fp8_unaligned_and_strided(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = _gen(6)
    m, n, k = 70, 90, 300
    A, SA, B, SB = _dense(g, m, n, k, 0, 1, 1, 128, wide=False)
    ref = (_spread(A, SA, 1, 128) @ _spread(B, SB, 128, 128)).float()
    C = torch.zeros(m, n, device="cuda")
    assert torch.equal(tb.matmul_fp8(A, SA, B, SB, C, beta=0), ref)
    # scales as strided views, operands cut from larger buffers at odd places
    sa = torch.zeros(_blocks(k), 2 * m, device="cuda").t()[::2]
    sa.copy_(SA)
    sb = torch.zeros(_blocks(n), _blocks(k) + 3, device="cuda")[:, 3:].t()
    sb.copy_(SB)
    a = torch.zeros(m + 1, k + 5, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)[1:, 5:]
    a.view(torch.uint8).copy_(A.view(torch.uint8))
    whole = torch.zeros(m, n + 3, device="cuda")
    tb.matmul_fp8(a, sa, B, sb, whole[:, 1:n + 1], beta=0)
    assert torch.equal(whole[:, 1:n + 1], ref) and not whole[:, 0].any() and not whole[:, n + 1:].any()
    # no rows, no columns, no k
    tb.matmul_fp8(A[:0], SA[:0], B, SB, C[:0])
    tb.matmul_fp8(A, SA, B[:, :0], SB[:, :0], C[:, :0])
    tb.matmul_fp8(A[:, :0], SA[:, :0], B[:0], SB[:0], C, beta=0)
    assert not C.any()


def test_fp8_nan_and_infinite_scales_stay_in_their_rows(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    A, SA, B, SB = _dense(_gen(7), 300, 2600, 256, 0, 1, 1, 128)
    clean = tb.matmul_fp8(A, SA, B, SB, torch.zeros(300, 2600, device="cuda"), beta=0)
    SA[17, 1] = float("nan")
    A.view(torch.uint8)[255, 3] = 0x7f
    got = tb.matmul_fp8(A, SA, B, SB, torch.zeros(300, 2600, device="cuda"), beta=0)
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[17] = bad[255] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])


def test_fp8_graph_and_streams(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = _gen(9)
    x = torch.randn(48, 1024, generator=g, device="cuda").bfloat16()
    w = torch.randn(512, 1024, generator=g, device="cuda").bfloat16()
    W, SW = tb.quantize_fp8(w, block=(128, 128))
    Q, S = tb.quantize_fp8(x)
    C = torch.zeros(48, 512, device="cuda")
    tb.matmul_fp8(Q, S, W.t(), SW.t(), C, beta=0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tb.quantize_fp8(x, Q, S)
        tb.matmul_fp8(Q, S, W.t(), SW.t(), C, beta=0)
    for i in range(3):
        x.copy_(torch.randn(48, 1024, generator=g, device="cuda"))
        graph.replay()
        got = C.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            q, sc = tb.quantize_fp8(x)
            again = tb.matmul_fp8(q, sc, W.t(), SW.t(), torch.zeros_like(C), beta=0)
        torch.cuda.synchronize()
        assert torch.equal(got, again)


def test_quantised_layer_and_its_gradients(cuda):
    """Y = X·W^T with both sides quantised, dX and dW from the gradient: each against the product of the values that
    the 8-bit operands stand for, and the whole against the unquantised product within the quantisation's error:
    e4m3 is off by at most 2^-4 relative (its least step below 2^-6 of the block's scale unit: 2^-10·S absolute)."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = _gen(21)
    m, n, k = 300, 264, 520
    X = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    W = (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)).bfloat16()
    D = torch.randn(m, n, generator=g, device="cuda").bfloat16()
    Qw, Sw = tb.quantize_fp8(W, block=(128, 128))

    def quant(x, per):
        q, s = tb.quantize_fp8(x, block=per)
        v = _spread(q, s, *per)
        slack = 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * _spread(torch.ones_like(x), s, *per)
        assert ((v - x.double()).abs() <= slack).all()
        return q, s, v, slack

    _, _, w, w_off = quant(W, (128, 128))

    def check(got, a, a_off, b, b_off, exact):
        # the product of the values themselves, as in test_matmul_fp8_real_values
        most = a.abs() @ b.abs()
        assert ((got.double() - a @ b).abs() <= (128 + 8) * 2.0 ** -23 * most + 2.0 ** -24 * most).all()
        off = a_off @ b.abs() + a.abs() @ b_off + a_off @ b_off
        assert ((got.double() - exact).abs() <= off + 1e-4 * most).all()

    q, s, x, x_off = quant(X, (1, 128))
    Y = tb.matmul_fp8(q, s, Qw.t(), Sw.t(), torch.zeros(m, n, device="cuda"), beta=0)
    check(Y, x, x_off, w.t(), w_off.t(), X.double() @ W.double().t())
    q, s, d, d_off = quant(D, (1, 128))
    dX = tb.matmul_fp8(q, s, Qw, Sw, torch.zeros(m, k, device="cuda"), beta=0)
    check(dX, d, d_off, w, w_off, D.double() @ W.double())
    qd, sd, d, d_off = quant(D, (128, 1))
    qx, sx, x, x_off = quant(X, (128, 1))
    dW = tb.matmul_fp8(qd.t(), sd.t(), qx, sx, torch.zeros(n, k, device="cuda"), beta=0)
    check(dW, d.t(), d_off.t(), x, x_off, D.double().t() @ X.double())


def test_expert_layer_together(cuda):
    """A mixture of experts as it is used: routed rows through two 8-bit products with a gate between, and the same
    layer in bf16 with its gradients, against autograd in 64 bits."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = _gen(30)
    E, tokens, top, k, h = 6, 150, 2, 256, 392
    x = torch.randn(tokens, k, generator=g, device="cuda").bfloat16()
    w1 = (torch.randn(E, h, k, generator=g, device="cuda") / math.sqrt(k)).bfloat16()
    w2 = (torch.randn(E, k, h, generator=g, device="cuda") / math.sqrt(h)).bfloat16()
    score = torch.randn(tokens, E, generator=g, device="cuda")
    score[:, 4] = -1e9  # an expert without rows
    expert = score.topk(top, dim=1).indices.flatten()
    order = torch.argsort(expert, stable=True)
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.bincount(expert, minlength=E).cumsum(0)
    rows = x[order // top].contiguous()
    R = tokens * top

    # bf16: forward, gradients of both weights and of the rows
    u = tb.grouped_matmul(rows, w1.transpose(1, 2), torch.empty(R, h, device="cuda"), off, beta=0)
    a = torch.relu(u).bfloat16()
    y = tb.grouped_matmul(a, w2.transpose(1, 2), torch.empty(R, k, device="cuda"), off, beta=0)
    dy = torch.randn(R, k, generator=g, device="cuda").bfloat16()
    dw2 = tb.grouped_matmul_wgrad(dy, a, torch.empty(E, k, h, device="cuda"), off, beta=0)
    da = tb.grouped_matmul(dy, w2, torch.empty(R, h, device="cuda"), off, beta=0)
    du = (da * (u > 0)).bfloat16()
    dw1 = tb.grouped_matmul_wgrad(du, rows, torch.empty(E, h, k, device="cuda"), off, beta=0)
    dx = tb.grouped_matmul(du, w1, torch.empty(R, k, device="cuda"), off, beta=0)
    ends = off.tolist()
    # each step against the formula on the step's own operands: exact products, k + 2 additions in f32
    def near(got, a, b, per):
        for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
            p, q = per(a, lo, hi, e), per(b, lo, hi, e)
            ref, most = p @ q, p.abs() @ q.abs()
            o = got[e] if got.dim() == 3 else got[lo:hi]
            assert ((o.double() - ref).abs() <= (p.shape[1] + 2) * 2.0 ** -23 * most).all()
    pick = lambda t, lo, hi, e: (t[e] if t.dim() == 3 else t[lo:hi]).double()
    near(u, rows, w1.transpose(1, 2), pick)
    near(y, a, w2.transpose(1, 2), pick)
    near(da, dy, w2, pick)
    near(dx, du, w1, pick)
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        for got, p, q in ((dw2, dy, a), (dw1, du, rows)):
            p, q = p[lo:hi].double().t(), q[lo:hi].double()
            assert ((got[e].double() - p @ q).abs() <= (hi - lo + 2) * 2.0 ** -23 * (p.abs() @ q.abs())).all()
    # the whole against autograd: bf16 roundings of a and du (2^-8 each) are all that is left
    t1, t2, tx = (t.double().requires_grad_() for t in (w1, w2, rows))
    outs = [torch.relu(tx[lo:hi] @ t1[e].t()) @ t2[e].t() for e, (lo, hi) in enumerate(zip(ends, ends[1:]))]
    torch.cat(outs).backward(dy.double())
    for got, ref in ((dw1, t1.grad), (dw2, t2.grad), (dx, tx.grad)):
        assert float((got.double() - ref).norm() / ref.norm()) <= 2.0 ** -8 + 1e-3
    assert not dw1[4].any() and not dw2[4].any()

    # 8 bits: quantise, multiply, gate, quantise, multiply
    q1, s1 = tb.quantize_fp8(w1, block=(128, 128))
    q2, s2 = tb.quantize_fp8(w2, block=(128, 128))
    qr, sr = tb.quantize_fp8(rows)
    u8 = tb.grouped_matmul_fp8(qr, sr, q1.transpose(1, 2), s1.transpose(1, 2), torch.empty(R, h, device="cuda"), off,
                               beta=0)
    qa, sa = tb.quantize_fp8(torch.relu(u8).bfloat16())
    y8 = tb.grouped_matmul_fp8(qa, sa, q2.transpose(1, 2), s2.transpose(1, 2), torch.empty(R, k, device="cuda"), off,
                               beta=0)
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        p, q = _spread(qr[lo:hi], sr[lo:hi], 1, 128), _spread(q1[e], s1[e], 128, 128).t()
        assert ((u8[lo:hi].double() - p @ q).abs() <= 140 * 2.0 ** -23 * (p.abs() @ q.abs())).all()
        p, q = _spread(qa[lo:hi], sa[lo:hi], 1, 128), _spread(q2[e], s2[e], 128, 128).t()
        assert ((y8[lo:hi].double() - p @ q).abs() <= 140 * 2.0 ** -23 * (p.abs() @ q.abs())).all()
    tb.device_status()


def test_scales_that_overlap_are_refused(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    X = torch.ones(4, 256, device="cuda")
    Q = torch.empty(4, 256, dtype=torch.float8_e4m3fn, device="cuda")
    with pytest.raises(tb.TBError, match="overlap"):
        tb.quantize_fp8(X, Q, torch.empty(4, 1, device="cuda").expand(4, 2))


@pytest.mark.parametrize("block", [(1, 128), (128, 1), (128, 128)])
def test_quantize_f32_off_the_nearest_only_at_borders(cuda, block):
    """0.4375·X is off by 2^-24 and the quotient by 2^-23 at most: where Q is not the nearest e4m3 value, it is the one
    on the other side of a border that lies within 2^-22 of the exact quotient."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    x = torch.randn(2048, 4096, generator=_gen(40), device="cuda")
    # quotients near a border: multiples of 1/16 of powers of two, a few f32 steps off
    x[:, ::2] = torch.ldexp(torch.randint(16, 32, (2048, 2048), generator=_gen(41), device="cuda").float() / 16,
                            torch.randint(-4, 5, (2048, 2048), generator=_gen(42), device="cuda"))
    x[:, ::2] *= 1 + 2.0 ** -23 * torch.randint(-3, 4, (2048, 2048), generator=_gen(43), device="cuda").float()
    x[::128, ::128] = 448.0 * (1 + 2.0 ** -20)
    Q, S = tb.quantize_fp8(x, block=block)
    q, s = _quantized64(x, *block)
    assert torch.equal(S, s.float())
    over = s.repeat_interleave(block[0], 0).repeat_interleave(block[1], 1)
    v, off = x.double() / over, Q.double() != q
    border = (Q.double() + q) / 2
    assert ((v - border).abs()[off] <= 2.0 ** -22 * v.abs()[off]).all()
