"""GPU: products of rows grouped by expert and their weight gradients,
against the formula in 64 bits.

Most inputs are small whole numbers: every product and every partial sum is
then exact in f32 (|sum| < 2^24), so the f32 output has to be equal, and a
16-bit output has to be the exact value rounded once."""
from __future__ import annotations

import itertools

import pytest

pytestmark = pytest.mark.gpu

OUT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def _types(name):
    import torch
    return getattr(torch, OUT[name])


def _ints(shape, g, dtype, most=3):
    import torch
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def _offsets(sizes, before=0, dtype=None):
    import torch
    ends = [before]
    for s in sizes:
        ends.append(ends[-1] + s)
    return torch.tensor(ends, dtype=dtype or torch.int32, device="cuda"), ends


def _reference(A, B, C, ends, beta):
    out = C.double().clone()
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        out[lo:hi] = A[lo:hi].double() @ B[e].double() + (out[lo:hi] if beta else 0)
    return out


# One shape for each kernel and the edges of each: (sizes of the groups, k, n)
SHAPES = {
    "one row": ([1], 8, 8),
    "one of everything": ([1], 1, 1),
    "empty groups": ([0, 3, 0, 0, 5, 0], 64, 64),
    "only empty": ([0, 0, 0], 64, 64),
    "decode": ([1, 0, 2, 1, 1, 0, 3, 1], 1024, 512),
    "decode, k ends inside a fill": ([2, 7, 1], 1000, 200),
    "33 rows": ([33, 31, 32], 256, 96),
    "odd widths": ([5, 130, 0, 127], 37, 51),
    "rows 96 and 97": ([96, 97, 128, 129], 136, 264),
    "128-wide tiles": ([100, 128, 60, 90, 128, 1, 77, 128], 192, 2432),
    "pair tiles": ([300, 0, 257, 700, 256, 487], 200, 2568),
    "pair tiles, many fills": ([512, 513, 511, 512], 1032, 2560),
    "many groups": ([i % 5 for i in range(300)], 72, 136),
}


@pytest.mark.parametrize("name", list(SHAPES))
@pytest.mark.parametrize("dtype,out,layout,beta", [("bf16", "f32", "kn", 1), ("f16", "f32", "nk", 0),
                                                   ("bf16", "bf16", "nk", 1), ("f16", "f16", "kn", 0)])
def test_grouped_matmul(cuda, name, dtype, out, layout, beta):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    sizes, k, n = SHAPES[name]
    g = torch.Generator(device="cuda")
    g.manual_seed(len(name) + k)
    dt = _types(dtype)
    before, behind = (3, 5) if len(sizes) > 1 else (0, 0)
    off, ends = _offsets(sizes, before, torch.int64 if beta else torch.int32)
    rows = ends[-1] + behind
    A = _ints((rows, k), g, dt)
    A[:before] = float("nan")            # rows of no group: never part of a result
    A[ends[-1]:] = float("inf")
    E = len(sizes)
    B = _ints((E, k, n), g, dt) if layout == "kn" else _ints((E, n, k), g, dt).transpose(1, 2)
    C = _ints((rows, n), g, _types(out), 7)
    ref = _reference(A, B, C, ends, beta)
    got = tb.grouped_matmul(A, B, C, off, beta=beta)
    tb.device_status()
    assert got is C
    assert torch.equal(C, ref.to(C.dtype))


@pytest.mark.parametrize("name", list(SHAPES))
@pytest.mark.parametrize("dtype,out,beta", [("bf16", "f32", 1), ("f16", "f16", 0), ("bf16", "bf16", 0)])
def test_grouped_matmul_wgrad(cuda, name, dtype, out, beta):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    sizes, k, n = SHAPES[name]
    if len(sizes) > 100:
        k, n = 24, 40
    g = torch.Generator(device="cuda")
    g.manual_seed(len(name) + n)
    dt = _types(dtype)
    before, behind = (3, 5) if len(sizes) > 1 else (0, 0)
    off, ends = _offsets(sizes, before)
    rows = ends[-1] + behind
    A, D = _ints((rows, k), g, dt, 2), _ints((rows, n), g, dt, 2)
    for t in (A, D):
        t[:before] = float("nan")
        t[ends[-1]:] = float("inf")
    G = _ints((len(sizes), k, n), g, _types(out), 7)
    ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
    if beta:
        ref += G.double()
    tb.grouped_matmul_wgrad(A, D, G, off, beta=beta)
    tb.device_status()
    assert torch.equal(G, ref.to(G.dtype))


@pytest.mark.parametrize("k,n", [(2304, 2560), (136, 264)])   # pair tiles, one-CTA tiles
def test_wgrad_every_length_inside_a_fill(cuda, k, n):
    """Groups of 64·j + r rows for every r, their neighbours' rows NaN and infinite."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    for r in range(0, 64, 7 if k > 1000 else 1):
        sizes = [64 + r, 3, r, 129]
        off, ends = _offsets(sizes, 1)
        A, D = _ints((ends[-1] + 2, k), g, torch.bfloat16, 2), _ints((ends[-1] + 2, n), g, torch.bfloat16, 2)
        A[ends[1]:ends[2]] = float("nan")  # group 1's gradient is NaN, its neighbours' are not
        D[ends[1]:ends[2]] = float("inf")
        G = torch.zeros(4, k, n, device="cuda")
        tb.grouped_matmul_wgrad(A, D, G, off, beta=0)
        for e in (0, 2, 3):
            ref = A[ends[e]:ends[e + 1]].double().t() @ D[ends[e]:ends[e + 1]].double()
            assert torch.equal(G[e], ref.float()), (r, e)
        assert torch.isnan(G[1]).all()
    tb.device_status()


@pytest.mark.parametrize("dtype,out,layout", list(itertools.product(["f16", "bf16"], ["f32", "f16", "bf16"], ["kn", "nk"])))
def test_real_values_round_once(cuda, dtype, out, layout):
    """|error| <= (k + 2)·2^-23·Σ|a||b| for k additions in f32, each off by at most one unit in the last place,
    and half a step of the output type for its rounding (f16 below 2^-14: half its least step, 2^-25)."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(11)
    dt, od = _types(dtype), _types(out)
    off, ends = _offsets([70, 0, 200, 41], 0)
    k, n = 520, 328
    A = torch.randn(ends[-1], k, generator=g, device="cuda").to(dt)
    B = torch.randn(4, k, n, generator=g, device="cuda").to(dt)
    if layout == "nk":
        B = B.transpose(1, 2).contiguous().transpose(1, 2)
    C = torch.randn(ends[-1], n, generator=g, device="cuda").to(od)
    ref = _reference(A, B, C, ends, 1)
    scale = _reference(A.abs(), B.abs(), C.abs(), ends, 1)
    tb.grouped_matmul(A, B, C, off)
    sums = (k + 2) * 2.0 ** -23 * scale
    tol = sums + torch.finfo(od).eps / 2 * (ref.abs() + sums) + 2.0 ** -25
    assert ((C.double() - ref).abs() <= tol).all()


def test_strided_and_unaligned_operands(cuda):
    """Views with a leading dimension, an odd base and transposed outputs' neighbours left alone."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    off, ends = _offsets([9, 0, 140, 3])
    rows, k, n = ends[-1], 72, 88
    for a_pad, a_skip, b_pad, c_skip in itertools.product([0, 8, 3], [0, 1, 8], [0, 5, 8], [0, 1, 4]):
        A = _ints((rows, k + a_pad + a_skip), g, torch.float16)[:, a_skip:a_skip + k]
        B = _ints((4, k + 1, n + b_pad), g, torch.float16)[:, :k, b_pad:]
        whole = _ints((rows, n + 2 * c_skip), g, torch.float32, 7)
        C = whole[:, c_skip:c_skip + n]
        want = whole.double().clone()
        want[:, c_skip:c_skip + n] = _reference(A, B, C, ends, 1)
        tb.grouped_matmul(A, B, C, off)
        assert torch.equal(whole.double(), want)
        G = torch.zeros(4, k, n + c_skip, device="cuda", dtype=torch.float32)
        D = _ints((rows, n + b_pad), g, torch.float16)[:, b_pad:]
        tb.grouped_matmul_wgrad(A, D, G[:, :, c_skip:], off)
        ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
        assert torch.equal(G[:, :, c_skip:].double(), ref)
        assert not G[:, :, :c_skip].any()
    tb.device_status()


def test_calls_like_an_earlier_one(cuda):
    """The same properties at other addresses, aligned or not, in turn with other layouts, types and beta."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(14)
    off, ends = _offsets([9, 0, 140, 3])
    rows, k, n = ends[-1], 72, 88
    for i in range(24):
        dt = (torch.float16, torch.bfloat16)[i % 2]
        buf = _ints((rows * k + 8,), g, dt)
        A = buf[(0, 8, 1, 3)[i % 4]:][:rows * k].view(rows, k)
        B = _ints((4, k, n), g, dt) if i % 3 else _ints((4, n, k), g, dt).transpose(1, 2)
        C = _ints((rows, n), g, (torch.float32, dt)[i // 12], 7)
        want = _reference(A, B, C, ends, i % 2).to(C.dtype)
        assert torch.equal(tb.grouped_matmul(A, B, C, off, beta=i % 2), want)
        D = _ints((rows, n), g, dt)
        G = _ints((4, k, n), g, torch.float32, 7)
        ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
        want = ref + (i % 2) * G.double()
        assert torch.equal(tb.grouped_matmul_wgrad(A, D, G, off, beta=i % 2).double(), want)
    with pytest.raises(tb.TBError, match="beta"):
        tb.grouped_matmul(A, B, C, off, beta=2)
    with pytest.raises(tb.TBError, match="disagree"):
        tb.grouped_matmul(A, B, C[1:], off)
    with pytest.raises(tb.TBError, match="entries"):
        tb.grouped_matmul(A, B, C, off[:-1])
    with pytest.raises(tb.TBError, match="both be"):
        tb.grouped_matmul(A.float(), B, C, off)
    with pytest.raises(tb.TBError, match="CUDA tensor"):
        tb.grouped_matmul(A, B, C, off.cpu())
    tb.device_status()


def test_threads(cuda):
    """Calls from two threads at once, each on a stream of its own."""
    import threading
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(15)
    off, ends = _offsets([90, 0, 33, 130])
    bad = []
    sets = [(_ints((ends[-1], k), g, torch.float16), _ints((4, k, 136), g, torch.float16)) for k in (64, 200)]
    torch.cuda.synchronize()

    def work(A, B):
        want = _reference(A, B, torch.zeros(ends[-1], 136, device="cuda"), ends, 0)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(50):
                C = tb.grouped_matmul(A, B, torch.zeros(ends[-1], 136, device="cuda"), off, beta=0)
                if not torch.equal(C.double(), want):
                    bad.append(A.shape)

    threads = [threading.Thread(target=work, args=s) for s in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_weights_in_interleaved_layouts(cuda):
    """B [groups, k, n] as a view of (k, groups, n) and of (n, groups, k) storage; G as a view of (k, groups, n)."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    off, ends = _offsets([40, 7, 0, 90])
    k, n = 80, 104
    A = _ints((ends[-1], k), g, torch.bfloat16)
    for B in (_ints((k, 4, n), g, torch.bfloat16).permute(1, 0, 2), _ints((n, 4, k), g, torch.bfloat16).permute(1, 2, 0)):
        C = torch.zeros(ends[-1], n, device="cuda")
        tb.grouped_matmul(A, B, C, off, beta=0)
        assert torch.equal(C.double(), _reference(A, B, C, ends, 0))
    D = _ints((ends[-1], n), g, torch.bfloat16)
    G = torch.zeros(k, 4, n, device="cuda").permute(1, 0, 2)
    tb.grouped_matmul_wgrad(A, D, G, off)
    ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
    assert torch.equal(G.double(), ref)


def test_no_rows_and_no_columns(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    h = dict(device="cuda", dtype=torch.float16)
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    C = torch.ones(4, 16, device="cuda")
    # k = 0: the rows of a group become beta·C, others stay
    tb.grouped_matmul(torch.empty(4, 0, **h), torch.empty(2, 0, 16, **h), C,
                      torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"), beta=0)
    assert torch.equal(C, torch.tensor([0., 0, 0, 1], device="cuda")[:, None].expand(4, 16))
    tb.grouped_matmul(torch.empty(0, 8, **h), torch.ones(2, 8, 16, **h), torch.empty(0, 16, device="cuda"), zero)
    tb.grouped_matmul(torch.ones(4, 8, **h), torch.ones(2, 8, 0, **h), torch.empty(4, 0, device="cuda"), zero)
    tb.grouped_matmul(torch.ones(4, 8, **h), torch.ones(0, 8, 16, **h), C, zero[:1])
    G = torch.ones(2, 8, 16, device="cuda")
    tb.grouped_matmul_wgrad(torch.empty(0, 8, **h), torch.empty(0, 16, **h), G, zero)
    assert (G == 1).all()
    tb.grouped_matmul_wgrad(torch.empty(0, 8, **h), torch.empty(0, 16, **h), G, zero, beta=0)
    assert not G.any()
    tb.device_status()


def test_offsets_outside_the_rows_are_clamped(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    A, B = _ints((50, 64), g, torch.float16), _ints((3, 64, 64), g, torch.float16)
    for bad in ([-9, 20, 30, 1 << 30], [-(1 << 31), 20, 30, 50]):
        C = torch.zeros(50, 64, device="cuda")
        tb.grouped_matmul(A, B, C, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        assert torch.equal(C.double(), _reference(A, B, C * 0, [0, 20, 30, 50], 0))
    C = torch.zeros(50, 64, device="cuda")   # a falling pair is an empty group
    tb.grouped_matmul(A, B, C, torch.tensor([10, 40, 5, 5], dtype=torch.int64, device="cuda"))
    assert torch.equal(C.double(), _reference(A, B, C * 0, [10, 40, 40, 40], 0))
    G = torch.zeros(3, 64, 64, device="cuda")
    tb.grouped_matmul_wgrad(A, A, G, torch.tensor([-5, 20, 30, 99], dtype=torch.int64, device="cuda"))
    ref = torch.stack([A[a:b].double().t() @ A[a:b].double() for a, b in ((0, 20), (20, 30), (30, 50))])
    assert torch.equal(G.double(), ref)
    tb.device_status()


def test_results_repeat_bit_for_bit(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    off, ends = _offsets([3, 1, 0, 4])
    A = torch.randn(8, 4096, generator=g, device="cuda").bfloat16()
    B = torch.randn(4, 4096, 512, generator=g, device="cuda").bfloat16()
    runs = [tb.grouped_matmul(A, B, torch.zeros(8, 512, device="cuda"), off).clone() for _ in range(5)]
    assert all(torch.equal(r, runs[0]) for r in runs)


def test_a_captured_graph_follows_the_offsets(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(10)
    rows, k, n = 400, 136, 200
    A, B = _ints((rows, k), g, torch.bfloat16), _ints((4, k, n), g, torch.bfloat16)
    D = _ints((rows, n), g, torch.bfloat16, 2)
    C, G = torch.zeros(rows, n, device="cuda"), torch.zeros(4, k, n, device="cuda")
    off, _ = _offsets([100, 100, 100, 100])
    tb.grouped_matmul(A, B, C, off, beta=0)
    tb.grouped_matmul_wgrad(A, D, G, off, beta=0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tb.grouped_matmul(A, B, C, off, beta=0)
        tb.grouped_matmul_wgrad(A, D, G, off, beta=0)
    for sizes in ([1, 0, 399, 0], [0, 0, 0, 400], [130, 5, 65, 200]):
        new, ends = _offsets(sizes)
        off.copy_(new)
        C.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(C.double(), _reference(A, B, torch.zeros_like(C), ends, 0))
        ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
        assert torch.equal(G.double(), ref)


def test_streams(cuda):
    """Two calls at once on two streams, one of them with repacked operands."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(12)
    off, ends = _offsets([200, 33, 0, 90])
    sets = []
    for k in (136, 137):
        A, B = _ints((ends[-1], k), g, torch.float16), _ints((4, k, 264), g, torch.float16)
        sets.append((A, B, torch.zeros(ends[-1], 264, device="cuda")))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (A, B, C), s in zip(sets, streams):
            tb.grouped_matmul(A, B, C, off, beta=0, stream=s)
    torch.cuda.synchronize()
    for A, B, C in sets:
        assert torch.equal(C.double(), _reference(A, B, C, ends, 0))


def test_gradients_against_the_formula_and_differences(cuda):
    """L = Σ W·C for C = grouped(A, B): dA and dB from the operators against the formula in 64 bits and against
    differences of L, which is linear in A and in B, so that a difference quotient has no error but rounding.
    Whole numbers: everything is exact."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(13)
    off, ends = _offsets([20, 0, 150, 7])
    k, n = 96, 80
    A, B = _ints((ends[-1], k), g, torch.bfloat16, 2), _ints((4, k, n), g, torch.bfloat16, 2)
    W = _ints((ends[-1], n), g, torch.bfloat16, 2)
    dA = torch.zeros(ends[-1], k, device="cuda")
    dB = torch.zeros(4, k, n, device="cuda")
    tb.grouped_matmul(W, B.transpose(1, 2), dA, off, beta=0)
    tb.grouped_matmul_wgrad(A, W, dB, off, beta=0)
    a, b = A.double().requires_grad_(), B.double().requires_grad_()
    loss = sum(((a[lo:hi] @ b[e]) * W[lo:hi].double()).sum() for e, (lo, hi) in enumerate(zip(ends, ends[1:])))
    loss.backward()
    assert torch.equal(dA.double(), a.grad) and torch.equal(dB.double(), b.grad)

    def value(A, B):
        C = torch.zeros(ends[-1], n, device="cuda")
        tb.grouped_matmul(A, B, C, off, beta=0)
        return (C.double() * W.double()).sum()

    base = value(A, B)
    for r, c in ((0, 0), (19, 95), (20, 3), (176, 50)):
        moved = A.clone()
        moved[r, c] += 1
        assert value(moved, B) - base == dA[r, c].double()
    for e, i, j in ((0, 0, 0), (1, 4, 4), (2, 95, 79), (3, 50, 1)):
        moved = B.clone()
        moved[e, i, j] += 1
        assert value(A, moved) - base == dB[e, i, j].double()


@pytest.mark.parametrize("sizes,k,n", [([4099], 136, 120), ([2000, 0, 1, 3000], 72, 256), ([515, 512, 510], 128, 128)])
def test_wgrad_of_few_tiles_over_many_rows(cuda, sizes, k, n):
    """K ranges shared by the CTAs of a cluster, ending inside a fill."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(16)
    off, ends = _offsets(sizes, 2)
    A, D = _ints((ends[-1] + 9, k), g, torch.bfloat16, 2), _ints((ends[-1] + 9, n), g, torch.bfloat16, 2)
    A[ends[-1]:] = float("nan")
    for out, beta in ((torch.float32, 1), (torch.bfloat16, 0)):
        G = _ints((len(sizes), k, n), g, out, 7)
        ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
        want = (ref + beta * G.double()).to(out)
        tb.grouped_matmul_wgrad(A, D, G, off, beta=beta)
        assert torch.equal(G, want)
    tb.device_status()


def test_more_elements_than_32_bits_count(cuda):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(17)
    rows, k, n = 270_000, 64, 8192   # C: 2.2e9 elements
    A, B = _ints((rows, k), g, torch.float16), _ints((3, k, n), g, torch.float16)
    off, ends = _offsets([5, 269_500, 300], 100)
    C = torch.full((rows, n), 3.0, device="cuda", dtype=torch.float16)
    tb.grouped_matmul(A, B, C, off, beta=0)
    for lo, hi, e in ((100, 105, 0), (200, 300, 1), (269_400, 269_605, 1), (269_605, 269_905, 2)):
        assert torch.equal(C[lo:hi].double(), A[lo:hi].double() @ B[e].double())
    assert (C[269_905:] == 3).all() and (C[:100] == 3).all()
    G = torch.zeros(3, k, n, device="cuda")
    tb.grouped_matmul_wgrad(A, C, G, off)
    for e in (0, 2):
        assert torch.equal(G[e].double(), A[ends[e]:ends[e + 1]].double().t() @ C[ends[e]:ends[e + 1]].double())
    tb.device_status()


def test_calls_follow_the_work_before_them(cuda):
    """Operands written by the kernel just before, outputs read by the one just after, without a wait between."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(18)
    off, ends = _offsets([3, 0, 200, 40])
    k = 256
    A, W = torch.zeros(ends[-1], k, device="cuda", dtype=torch.bfloat16), _ints((4, k, k), g, torch.bfloat16, 1)
    values = [_ints((ends[-1], k), g, torch.bfloat16, 1) for _ in range(6)]
    C, out = torch.zeros(ends[-1], k, device="cuda"), []
    for i in range(60):
        A.copy_(values[i % 6])
        tb.grouped_matmul(A, W, C, off, beta=0)
        Q, S = tb.quantize_fp8(C)
        out.append((C.clone(), Q.float() * S.repeat_interleave(128, 1)))
    for i, (c, v) in enumerate(out):
        assert torch.equal(c.double(), _reference(values[i % 6], W, torch.zeros_like(c), ends, 0))
        # e4m3: off by at most 2^-4 relative, and half its least step (2^-10) in units of the scale below that
        assert ((v - c).abs() <= 2.0 ** -4 * c.abs() + 2.0 ** -10 * c.abs().amax() / 448).all()


def test_offsets_that_fall_and_rise_stay_inside(cuda):
    """Rows in several groups: every group has the same weights, so that each gives the same rows."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(10)
    A, B = _ints((300, 64), g, torch.float16), _ints((1, 64, 64), g, torch.float16)
    C = torch.full((302, 64), 7.0, device="cuda")
    off = torch.tensor([0, 300] * 20 + [0], dtype=torch.int32, device="cuda")   # 20 groups of all rows among 40
    tb.grouped_matmul(A, B.repeat(40, 1, 1), C[1:301], off, beta=0)
    assert torch.equal(C[1:301].double(), A.double() @ B[0].double())
    assert (C[0] == 7).all() and (C[301] == 7).all()
    tb.device_status()


@pytest.mark.parametrize("beta", [0.5, 2, -1, None])
def test_beta_is_zero_or_one(cuda, beta):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    A, B = torch.ones(4, 64, device="cuda").half(), torch.ones(1, 64, 64, device="cuda").half()
    off, C = torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.ones(4, 64, device="cuda")
    for _ in range(2):   # 1.0 and True are 1
        tb.grouped_matmul(A, B, C, off, beta=1.0)
        tb.grouped_matmul(A, B, C, off, beta=True)
        with pytest.raises(tb.TBError, match="beta"):
            tb.grouped_matmul(A, B, C, off, beta=beta)
    assert (C == 257).all()


@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("eight_bit", [False, True])
def test_outputs_off_vector_boundaries(cuda, eight_bit, out):
    """Rows that begin anywhere, widths that end anywhere: the places beside the output keep what they held."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(16)
    dt = getattr(torch, out)
    off, ends = _offsets([3, 0, 130, 33])
    rows, k = ends[-1], 128
    A = _ints((rows, k), g, torch.float16, 2)
    for n, skip, pad, beta in itertools.product([1, 2, 31, 33, 64, 95, 130, 383], [0, 1, 2, 3], [0, 1, 2], [0, 1]):
        whole = _ints((rows + 1, skip + n + pad), g, dt, 7)
        C, want = whole[:rows, skip:skip + n], whole.clone()
        B = _ints((4, k, n), g, torch.float16, 2)
        want[:rows, skip:skip + n] = _reference(A, B, C, ends, beta).to(dt)
        if eight_bit:
            one = torch.ones(rows, 1, device="cuda")
            f8 = torch.float8_e4m3fn
            SB = torch.ones(4, 1, n if n % 2 else (n + 127) // 128, device="cuda")
            tb.grouped_matmul_fp8(A.to(f8), one, B.to(f8), SB, C, off, beta=beta)
        else:
            tb.grouped_matmul(A, B, C, off, beta=beta)
        assert torch.equal(whole, want), (n, skip, pad, beta)
    tb.device_status()


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_weight_gradients_off_vector_boundaries(cuda, out):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(17)
    dt = getattr(torch, out)
    off, ends = _offsets([3, 0, 130, 33])
    A = _ints((ends[-1], 300), g, torch.float16, 2)
    for n, pad, beta in itertools.product([33, 257, 511], [0, 1], [0, 1]):
        D = _ints((ends[-1], n), g, torch.float16, 2)
        whole = _ints((4, 300, n + pad), g, dt, 7)
        G, want = whole[:, :, pad:], whole.clone()
        ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
        want[:, :, pad:] = (ref + beta * G.double()).to(dt)
        tb.grouped_matmul_wgrad(A, D, G, off, beta=beta)
        assert torch.equal(whole, want), (n, pad, beta)
    tb.device_status()


def test_repacked_calls_again(cuda):
    """Operands off 16-byte boundaries, the second time like the first: another stream, a graph, a workspace of one's own."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(18)
    off, ends = _offsets([9, 0, 140, 3])
    A, B = _ints((ends[-1], 77), g, torch.float16), _ints((4, 77, 51), g, torch.float16)
    C = torch.zeros(ends[-1], 51, device="cuda")
    want = _reference(A, B, C, ends, 0).float()
    for _ in range(3):
        tb.grouped_matmul(A, B, C, off, beta=0)
    assert torch.equal(C, want)
    with pytest.raises(tb.TBError, match="workspace"):
        tb.grouped_matmul(A, B, C, off, beta=0, workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        C2 = torch.zeros_like(C)
        for _ in range(3):
            tb.grouped_matmul(A, B, C2, off, beta=1)
    side.synchronize()
    assert torch.equal(C2, 3 * want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tb.grouped_matmul(A, B, C, off, beta=1)
        tb.grouped_matmul_wgrad(A, C2.half(), torch.zeros(4, 77, 51, device="cuda"), off, beta=0)
    A.copy_(_ints(tuple(A.shape), g, torch.float16))
    want = C.double() + _reference(A, B, C, ends, 0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(C.double(), want)
    tb.device_status()


# (groups, n, k, output, 8 bits): several tiles to a cluster of 2, 4 or 8 CTAs that share each tile's K range
SHARED = [(32, 1408, 2048, "f16", False), (10, 4096, 1024, "bf16", False), (24, 2048, 4096, "f32", False),
          (5, 2048, 4096, "f32", False), (5, 2048, 8192, "bf16", True)]


@pytest.mark.parametrize("groups,n,k,out,eight_bit", SHARED)
@pytest.mark.parametrize("rows", [1, 3, 7, 33, 39])
def test_shared_tiles_of_fewer_rows_than_ctas(cuda, groups, n, k, out, eight_bit, rows):
    """Tiles, and last blocks of 32 rows, with fewer rows than the cluster has CTAs, one after another: a CTA without
    a row may not run ahead of the others."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(19)
    off, ends = _offsets([max(1, rows - e % 3) for e in range(groups)])
    A, B = _ints((ends[-1], k), g, torch.float16, 2), _ints((groups, n, k), g, torch.float16, 2).transpose(1, 2)
    C = _ints((ends[-1], n), g, _types(out), 7)
    want = [_reference(A, B, C, ends, beta).to(C.dtype) for beta in (0, 1)]
    if eight_bit:
        f8 = torch.float8_e4m3fn
        A, B = A.to(f8), B.to(f8)
        SA, SB = torch.ones(ends[-1], k // 128, device="cuda"), torch.ones(groups, k // 128, n // 128, device="cuda")
    for i in range(40):
        got = C.clone()
        if eight_bit:
            tb.grouped_matmul_fp8(A, SA, B, SB, got, off, beta=i % 2)
        else:
            tb.grouped_matmul(A, B, got, off, beta=i % 2)
        assert torch.equal(got, want[i % 2]), i
    tb.device_status()


@pytest.mark.parametrize("groups,k,n,rows", [(64, 1, 384, 1024), (64, 33, 384, 1024), (100, 3, 384, 1024),
                                             (40, 3, 256, 4096)])
def test_shared_weight_gradients_of_fewer_rows_than_ctas(cuda, groups, k, n, rows):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(20)
    off, ends = _offsets([rows + e % 5 for e in range(groups)])
    A, D = _ints((ends[-1], (k + 7) // 8 * 8), g, torch.bfloat16, 2)[:, :k], _ints((ends[-1], n), g, torch.bfloat16, 2)
    G = _ints((groups, k, n), g, torch.float32, 7)
    ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
    for i in range(40):
        got = G.clone()
        tb.grouped_matmul_wgrad(A, D, got, off, beta=i % 2)
        assert torch.equal(got.double(), ref + i % 2 * G.double()), i
    tb.device_status()


@pytest.mark.parametrize("m", [33, 35, 39])
def test_shared_8_bit_tiles_of_one_matrix(cuda, m):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(21)
    A, B = _ints((m, 4096), g, torch.float16, 2), _ints((4096, 4096), g, torch.float16, 2)
    want = (A.double() @ B.double()).float()
    f8, one = torch.float8_e4m3fn, torch.ones(m, 32, device="cuda")
    A, B = A.to(f8), B.t().contiguous().to(f8).t()
    for _ in range(40):
        C = tb.matmul_fp8(A, one, B, torch.ones(32, 32, device="cuda"), torch.zeros(m, 4096, device="cuda"), beta=0)
        assert torch.equal(C, want)
    tb.device_status()


# Sums of one sign: truncated additions would all lean the same way.
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_weight_gradients_round_once(cuda, dtype):
    """Four million rows. A segment of 512 of them is off by at most 2^-23 per element, the f32 sums of the segments
    by 2^-24 each (a CTA of a cluster has an eighth of them at least, the eight are added at the end), then half a step
    of the output."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(22)
    rows, k, n, dt = 1 << 22, 64, 72, _types(dtype)
    A = torch.rand(rows, k, generator=g, device="cuda").to(dt)
    D = (torch.rand(rows, n, generator=g, device="cuda") / 128).to(dt)
    off = torch.tensor([0, 5, rows], dtype=torch.int32, device="cuda")
    G = tb.grouped_matmul_wgrad(A, D, torch.zeros(2, k, n, device="cuda", dtype=dt), off, beta=0)
    tb.device_status()
    for e, (lo, hi) in enumerate(((0, 5), (5, rows))):
        ref = torch.zeros(k, n, device="cuda", dtype=torch.float64)
        for at in range(lo, hi, 1 << 20):
            ref += A[at:min(hi, at + (1 << 20))].double().t() @ D[at:min(hi, at + (1 << 20))].double()
        sums = (512 * 2.0 ** -23 + (rows // 512 + 8) * 2.0 ** -24) * ref
        tol = sums + torch.finfo(dt).eps / 2 * (ref + sums)
        assert ((G[e].double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("sizes,n", [([3, 2], 256), ([300, 257], 2568)])   # shared tiles, pair tiles
def test_long_k_rounds_once(cuda, dtype, sizes, n):
    """As the gradients above, k = 65536 (16384 for the larger): segments of 512 elements."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(23)
    k, dt = 65536 if n < 1000 else 16384, _types(dtype)
    off, ends = _offsets(sizes)
    A = torch.rand(ends[-1], k, generator=g, device="cuda").to(dt)
    B = (torch.rand(2, k, n, generator=g, device="cuda") / 16).to(dt)
    C = tb.grouped_matmul(A, B, torch.zeros(ends[-1], n, device="cuda", dtype=dt), off, beta=0)
    tb.device_status()
    ref = _reference(A, B, torch.zeros_like(C), ends, 0)
    sums = (512 * 2.0 ** -23 + (k // 512 + 8) * 2.0 ** -24) * ref
    assert ((C.double() - ref).abs() <= sums + torch.finfo(dt).eps / 2 * (ref + sums)).all()


def test_tiles_longer_than_a_second(cuda):
    """One group has 330 million of the rows of 1000 groups, a tile of more than a second: the waits for it, and those
    of the next call, which is on the SMs that the others left, go on. Whole numbers whose sums stay below 2^24."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(24)
    sizes = [330_000_005] + [e % 3 for e in range(999)]
    off, ends = _offsets(sizes)
    rows = ends[-1]
    A, D = (torch.empty(rows, 8, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    first = torch.zeros(8, 8, device="cuda", dtype=torch.float64)
    for at in range(0, rows, 1 << 24):
        end = min(rows, at + (1 << 24))
        for t in (A, D):
            t[at:end] = torch.randint(-2, 3, (end - at, 8), generator=g, device="cuda", dtype=torch.int8)
        in_first = min(end, ends[1])
        first += A[at:in_first].double().t() @ D[at:in_first].double()
    ref = torch.stack([first] + [A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends[1:], ends[2:])])
    few, few_ends = _offsets([5, 0, 130, 40])
    A2, B2 = _ints((175, 64), g, torch.bfloat16), _ints((4, 64, 128), g, torch.bfloat16)
    C2 = torch.zeros(175, 128, device="cuda")
    G = torch.zeros(1000, 8, 8, device="cuda")
    times = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    times[0].record()
    tb.grouped_matmul_wgrad(A, D, G, off, beta=0)
    tb.grouped_matmul(A2, B2, C2, few, beta=0)
    times[1].record()
    tb.device_status()
    assert times[0].elapsed_time(times[1]) > 1000
    assert torch.equal(G.double(), ref)
    assert torch.equal(C2.double(), _reference(A2, B2, torch.zeros_like(C2), few_ends, 0))


def test_expired_wait_is_reported(cuda):
    """A wait of these kernels that runs out: the status says so once, both status words are cleared, and the context
    stays usable."""
    import ctypes
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    from mini_triton_nvgpu_v1_b200 import _capi
    lib, raw = _capi.load(), ctypes.c_uint32()
    assert tb.device_status() == 0
    for both in (False, True):
        assert lib.tb_selftest_grouped_wait(None, 2_000_000) == 0       # ~1 ms of SM clocks
        if both:
            assert lib.tb_selftest_bounded_wait(None, 2_000_000) == 0
        assert lib.tb_device_status(None, ctypes.byref(raw)) == _capi.TB_ERR_DEVICE_TIMEOUT
        assert raw.value >> 16 == _capi.TB_ERR_DEVICE_TIMEOUT << 8 | 5   # the first wait that gave up
        assert tb.device_status() == 0
    off, ends = _offsets([3, 5])
    A, B = torch.ones(8, 64, device="cuda").half(), torch.ones(2, 64, 64, device="cuda").half()
    assert (tb.grouped_matmul(A, B, torch.zeros(8, 64, device="cuda"), off) == 64).all()
    assert tb.device_status() == 0


def test_outputs_that_share_storage_until_written(cuda):
    """A lazy clone as the output of a call like an earlier one: its source keeps what it held."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(25)
    off, ends = _offsets([9, 0, 30])
    A, B = _ints((39, 64), g, torch.bfloat16), _ints((3, 64, 128), g, torch.bfloat16)
    D = _ints((39, 128), g, torch.bfloat16)
    one, f8 = torch.ones(39, 1, device="cuda"), torch.float8_e4m3fn
    SB, W = torch.ones(3, 1, 1, device="cuda"), _ints((64, 128), g, torch.bfloat16)
    X = torch.randn(39, 128, generator=g, device="cuda")
    calls = {
        "rows": (lambda o: tb.grouped_matmul(A, B, *o, off), [torch.zeros(39, 128, device="cuda")]),
        "wgrad": (lambda o: tb.grouped_matmul_wgrad(A, D, *o, off), [torch.zeros(3, 64, 128, device="cuda")]),
        "quantize": (lambda o: tb.quantize_fp8(X, *o), [torch.zeros(39, 128, device="cuda").to(f8), torch.zeros(39, 1, device="cuda")]),
        "fp8": (lambda o: tb.matmul_fp8(A.to(f8), one, W.to(f8), SB[0], *o), [torch.zeros(39, 128, device="cuda")]),
        "rows fp8": (lambda o: tb.grouped_matmul_fp8(A.to(f8), one, B.to(f8), SB, *o, off), [torch.zeros(39, 128, device="cuda")]),
    }
    for name, (call, source) in calls.items():
        plain = [s.clone() for s in source]
        call(plain)
        for _ in range(2):
            lazy = [torch._lazy_clone(s) for s in source]
            call(lazy)
            assert not any(s.float().any() for s in source), name
            assert all(torch.equal(x.float(), y.float()) for x, y in zip(lazy, plain)), name
    tb.device_status()


@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("sizes,widths", [([3, 0, 130, 33], [1, 33, 130, 383]), ([300, 700, 1, 513], [2567, 2306])])
def test_outputs_of_segments_off_vector_boundaries(cuda, out, sizes, widths):
    """As test_outputs_off_vector_boundaries, K long enough for sums of segments; one-CTA tiles and pairs."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(26)
    dt, k = getattr(torch, out), 1100
    off, ends = _offsets(sizes, 1)
    rows = ends[-1] + 2
    A = torch.zeros(rows, 1104, device="cuda", dtype=torch.float16)[:, :k]
    A.copy_(_ints((rows, k), g, torch.float16, 1))
    for n, skip, pad, beta in itertools.product(widths, [0, 1, 3, 8], [0, 1, 2], [0, 1]):
        whole = _ints((rows + 1, skip + n + pad), g, dt, 7)
        C, want = whole[:rows, skip:skip + n], whole.clone()
        B = _ints((4, (n + 7) // 8 * 8, 1104), g, torch.float16, 1)[:, :n, :k].transpose(1, 2)
        want[:rows, skip:skip + n] = _reference(A, B, C, ends, beta).to(dt)
        tb.grouped_matmul(A, B, C, off, beta=beta)
        assert torch.equal(whole, want), (n, skip, pad, beta)
    tb.device_status()


@pytest.mark.parametrize("out", ["float32", "float16"])
def test_weight_gradients_of_segments_off_vector_boundaries(cuda, out):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(27)
    dt = getattr(torch, out)
    for (k, sizes), n, pad, beta in itertools.product([(72, [3, 0, 1300, 33]), (1000, [1100, 7, 0, 1500])], [33, 257, 2049],
                                                      [0, 1], [0, 1]):
        off, ends = _offsets(sizes)
        A = _ints((ends[-1], k), g, torch.float16, 1)
        D = _ints((ends[-1], (n + 7) // 8 * 8), g, torch.float16, 1)[:, :n]
        whole = _ints((4, k, n + pad), g, dt, 7)
        G, want = whole[:, :, pad:], whole.clone()
        ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
        want[:, :, pad:] = (ref + beta * G.double()).to(dt)
        tb.grouped_matmul_wgrad(A, D, G, off, beta=beta)
        assert torch.equal(whole, want), (k, n, pad, beta)
    tb.device_status()


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("sizes,n,k", [([100, 1, 2], 2048, 1024), ([8, 8, 8], 2048, 1024), ([130, 70], 2048, 1024),
                                       ([1000] + [0] * 7, 1001, 1024), ([120, 3, 2, 3], 2048, 4096), ([120, 70, 2], 2048, 8192),
                                       ([100] + [1] * 23, 2048, 4096), ([1] * 12 + [128] + [2] * 11, 2048, 4096)])
def test_shared_tiles_of_uneven_groups(cuda, sizes, n, k, out):
    """Tiles of more rows than are exchanged at a time, before and behind tiles of fewer."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(28)
    off, ends = _offsets(sizes)
    A, B = _ints((ends[-1], k), g, torch.bfloat16, 2), _ints((len(sizes), n, k), g, torch.bfloat16, 2).transpose(1, 2)
    C = _ints((ends[-1], n), g, _types(out), 7)
    want = [_reference(A, B, C, ends, beta).to(C.dtype) for beta in (0, 1)]
    for i in range(40):
        got = C.clone()
        tb.grouped_matmul(A, B, got, off, beta=i % 2)
        assert torch.equal(got, want[i % 2]), i
    tb.device_status()


@pytest.mark.parametrize("groups,k,n,rows", [(8, 100, 1408, 2500), (100, 70, 384, 4000), (12, 128, 128, 3000)])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_shared_weight_gradients_of_many_rows(cuda, groups, k, n, rows, out):
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(29)
    off, ends = _offsets([rows + 7 * e % 11 for e in range(groups)])
    A, D = _ints((ends[-1], (k + 7) // 8 * 8), g, torch.float16, 2)[:, :k], _ints((ends[-1], n), g, torch.float16, 2)
    G = _ints((groups, k, n), g, _types(out), 7)
    ref = torch.stack([A[lo:hi].double().t() @ D[lo:hi].double() for lo, hi in zip(ends, ends[1:])])
    want = [ref.to(G.dtype), (ref + G.double()).to(G.dtype)]
    for i in range(40):
        got = G.clone()
        tb.grouped_matmul_wgrad(A, D, got, off, beta=i % 2)
        assert torch.equal(got, want[i % 2]), i
    tb.device_status()


def test_two_graphs_at_once(cuda):
    """Two captured graphs of calls that repack their operands and share tiles, replayed on two streams at once."""
    import torch
    import mini_triton_nvgpu_v1_b200 as tb
    g = torch.Generator(device="cuda")
    g.manual_seed(30)
    off, ends = _offsets([9, 0, 40, 3])
    sets = []
    for k in (1025, 2047):
        A, B = _ints((ends[-1], k), g, torch.float16, 2), _ints((4, k, 520), g, torch.float16, 2)
        C = torch.zeros(ends[-1], 520, device="cuda")
        tb.grouped_matmul(A, B, C, off, beta=0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(3):
                tb.grouped_matmul(A, B, C, off, beta=0)
        sets.append((A, B, C, graph, torch.cuda.Stream()))
    for _ in range(20):
        for A, B, C, graph, s in sets:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for A, B, C, _, _ in sets:
        assert torch.equal(C.double(), _reference(A, B, torch.zeros_like(C), ends, 0))
    tb.device_status()
