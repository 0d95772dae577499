"""Products with 4-bit weights (nestquant_b200.w4) against the definition in 64 bits.

Tolerance: q - zero times x is exact; a sum of K such products in 32 bits goes through at most 2 x 8 additions of a group on the tensor pipe, one per
group and chunk and a few between warps, each off by at most 2^-23 (truncation) of the sum of the terms' magnitudes; then half a step of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(N, K, g, dtype=F16, zeros=True, E=None, seed=1):
    gen = torch.Generator("cuda").manual_seed(seed)
    lead = () if E is None else (E,)
    q = torch.randint(0, 256, lead + (N, K // 2), generator=gen, device="cuda", dtype=torch.uint8)
    s = (0.01 * torch.randn(lead + (N, K // g), generator=gen, device="cuda")).to(dtype)
    z = torch.randint(0, 16, lead + (N, K // g), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    return q, s, z


def dense(q, s, z, g):
    n = torch.stack([q & 15, q >> 4], -1).flatten(-2).double()
    z = 8.0 if z is None else z.double().repeat_interleave(g, -1)
    return (n - z) * s.double().repeat_interleave(g, -1)


def check(got, x, w, K):
    """got = x W^T for rows that one matrix has"""
    x = x.double()
    want, size = x @ w.T, x.abs() @ w.abs().T
    n = 2 * 8 + K // 32 + K // 128 + 16
    tol = n * 2.0 ** -23 * size + torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 1e-6) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), got.shape, got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("T", [1, 2, 8, 9, 33])
@pytest.mark.parametrize("N,K,g,dtype,sdtype,out,zeros", [
    (16, 128, 128, F16, F16, F16, False), (1, 32, 32, F16, F16, F32, True), (40, 96, 32, BF16, BF16, BF16, True), (17, 320, 64, F16, BF16, F16, True),
    (100, 1024, 64, BF16, F16, F32, False), (513, 640, 128, BF16, BF16, BF16, True), (256, 2048, 32, F16, F16, F32, True), (130, 6144, 128, F16, F16, F16, True),
])
def test_products_match_the_definition(T, N, K, g, dtype, sdtype, out, zeros):
    from nestquant_b200 import w4
    q, s, z = make(N, K, g, sdtype, zeros, seed=N + T)
    x = torch.randn(T, K, generator=torch.Generator("cuda").manual_seed(T), device="cuda").to(dtype)
    y = w4.W4(q, s, z)(x, dtype=out)
    assert y.shape == (T, N) and y.dtype == out
    check(y, x, dense(q, s, z, g), K)


@pytest.mark.parametrize("T", [63, 64, 65, 127, 129, 300, 512, 1000])
@pytest.mark.parametrize("N,K,g,dtype,out,zeros", [(272, 1024, 128, F16, F16, True), (100, 608, 32, BF16, F32, False), (384, 448, 64, BF16, BF16, True), (129, 128, 128, F16, F32, False)])
def test_many_rows(T, N, K, g, dtype, out, zeros):
    from nestquant_b200 import w4
    q, s, z = make(N, K, g, dtype, zeros, seed=N + T)
    x = torch.randn(T, K, generator=torch.Generator("cuda").manual_seed(T), device="cuda").to(dtype)
    check(w4.W4(q, s, z)(x, dtype=out), x, dense(q, s, z, g), K)


def test_every_weight_of_a_unit_is_in_its_place():
    """one-hot rows: the results are the columns of the matrix, exactly"""
    from nestquant_b200 import w4
    for g in (32, 64, 128):
        for dtype in (F16, BF16):
            q, s, z = make(48, 384, g, dtype, True, seed=g)
            s = torch.full_like(s, 0.5)
            y = w4.W4(q, s, z)(torch.eye(384, device="cuda", dtype=dtype), dtype=F32)
            assert torch.equal(y.double().T, dense(q, s, z, g))


def rows_of(sizes, E, extra=0):
    start = torch.tensor([0] + list(sizes), dtype=torch.int32).cumsum(0).int().cuda()
    assert start.numel() == E + 1
    return start, int(start[-1]) + extra


@pytest.mark.parametrize("sizes,extra", [([0, 0, 0, 0, 0], 0), ([0, 0, 0, 0, 0], 3), ([1, 0, 2, 0, 1], 0), ([5, 8, 9, 0, 33], 7), ([0, 0, 0, 70, 0], 1), ([16, 17, 1, 3, 32], 40), ([30, 40, 20, 31, 29], 2), ([200, 1, 130, 0, 64], 0), ([30], 5), ([3], 40), ([500], 0)])
@pytest.mark.parametrize("N,K,g,dtype,out,zeros", [(48, 256, 128, F16, F16, False), (100, 352, 32, BF16, F32, True), (257, 1024, 64, BF16, BF16, True)])
def test_a_matrix_per_expert(sizes, extra, N, K, g, dtype, out, zeros):
    from nestquant_b200 import w4
    E = len(sizes)
    q, s, z = make(N, K, g, dtype, zeros, E=E, seed=N)
    start, P = rows_of(sizes, E, extra)
    x = torch.randn(P, K, generator=torch.Generator("cuda").manual_seed(P), device="cuda").to(dtype)
    y = w4.W4(q, s, z)(x, start=start, dtype=out)
    assert y.shape == (P, N)
    for e in range(E):
        a, b = int(start[e]), int(start[e + 1])
        if a < b:
            check(y[a:b], x[a:b], dense(q[e], s[e], None if z is None else z[e], g), K)
    assert (y[int(start[-1]):] == 0).all()


@pytest.mark.parametrize("dtype,g", [(F16, 128), (BF16, 32)])
def test_the_number_of_rows_is_the_devices(dtype, g):
    """a captured call whose start array has few rows, then many, then none, then one that falls: whichever form of the product takes it, rows behind are zero"""
    from nestquant_b200 import w4
    E, N, K, P = 5, 100, 384, 90
    q, s, z = make(N, K, g, dtype, True, E=E, seed=3)
    w = w4.W4(q, s, z)
    x = torch.randn(P, K, generator=torch.Generator("cuda").manual_seed(8), device="cuda").to(dtype)
    start = rows_of([1, 2, 3, 0, 1], E)[0]
    w(x, start=start)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = w(x, start=start, dtype=F32)
    for sizes in ([1, 2, 3, 0, 1], [10, 8, 0, 13, 9], [9, 0, 31, 0, 1], [18, 18, 18, 18, 18], [0, 0, 0, 0, 0], [0, 0, 39, 1, 0], [90, 0, 0, 0, 0], [0, 0, 0, 0, 7]):
        start.copy_(rows_of(sizes, E)[0])
        y.fill_(float("nan"))
        graph.replay()
        for e in range(E):
            a, b = int(start[e]), int(start[e + 1])
            if a < b:
                check(y[a:b], x[a:b], dense(q[e], s[e], z[e], g), K)
        assert (y[int(start[-1]):] == 0).all(), sizes
    for last in (30, 60, -2 ** 31):
        start.copy_(torch.tensor([0, 9, 8, 12, 20, last], dtype=torch.int32))
        y.fill_(float("nan"))
        graph.replay()
        assert (y == 0).all()


def test_the_number_of_rows_is_the_devices_with_64_mb_of_planes():
    """likewise, where calls of few rows an expert have a form of their own between the smallest and the call's bound"""
    from nestquant_b200 import w4
    E, N, K, g, P = 64, 1024, 2048, 64, 64 * 45
    q, s, z = make(N, K, g, F16, False, E=E, seed=3)
    w = w4.W4(q, s)
    x = torch.randn(P, K, generator=torch.Generator("cuda").manual_seed(8), device="cuda").half()
    start = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    w(x, start=start)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = w(x, start=start, dtype=F32)
    gen = torch.Generator().manual_seed(1)
    for total in (0, 1, 512, 513, 1365, 1366, P - 1, P):        # 8 and 64 / 3 rows an expert, and one more
        cuts = torch.cat([torch.zeros(1), torch.randint(0, total + 1, (E - 1,), generator=gen).sort()[0], torch.full((1,), total)]).int()
        start.copy_(cuts)
        y.fill_(float("nan"))
        graph.replay()
        for e in range(E):
            a, b = int(cuts[e]), int(cuts[e + 1])
            if a < b:
                check(y[a:b], x[a:b], dense(q[e], s[e], None, g), K)
        assert (y[total:] == 0).all(), total


def test_a_rows_bits_do_not_depend_on_the_others_in_its_call():
    """at the sizes of a decode call: the order of a row's sums goes by the matrix alone"""
    from nestquant_b200 import w4
    q, s, z = make(256, 1024, 64)
    w = w4.W4(q, s, z)
    x = torch.randn(8, 1024, device="cuda").half()
    y = w(x)
    assert torch.equal(w(x), y) and torch.equal(w(x.clone()), y)
    assert torch.equal(w(x[3:4].contiguous()), w(x[3:4].expand(1, 1024)))


def test_strided_and_unaligned_rows():
    from nestquant_b200 import w4
    q, s, z = make(40, 128, 64)
    w, W = w4.W4(q, s, z), dense(q, s, z, 64)
    buf = torch.randn(60, 300, device="cuda").half()
    for x in (buf[:9, :128], buf[:9, 8:136], buf[:9, 3:131], buf[::5, 16:144], buf.t()[:20, :128] if buf.shape[0] >= 128 else buf[:, :128], buf[:1, :128].expand(5, 128), buf[4:5, 1:129]):
        check(w(x), x, W, 128)
    assert w(buf[:0, :128]).shape == (0, 40)
    odd = torch.empty(q.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(q.shape).copy_(q)      # weights off two bytes, strided scales
    wide = torch.empty(40, 6, dtype=s.dtype, device="cuda")
    wide[:, ::3] = s
    x = buf[:9, :128]
    assert torch.equal(w4.W4(odd, wide[:, ::3], z.t().contiguous().t())(x), w(x))


def test_values_that_are_not_finite_stay_in_their_rows():
    from nestquant_b200 import w4
    q, s, z = make(64, 256, 128, zeros=False)
    q[5] = 0x99                                    # 9 - 8 = 1
    s[7, 1] = float("inf")
    w, x = w4.W4(q, s, z), torch.randn(12, 256, device="cuda").half()
    clean = w(x)
    x[3, 17] = float("inf")
    x[4, 200] = float("nan")
    y = w(x)
    keep = [r for r in range(12) if r not in (3, 4)]
    assert torch.equal(y[keep].nan_to_num(), clean[keep].nan_to_num()) and y[4].isnan().all() and y[3, 5] == float("inf")
    assert not y[keep][:, [n for n in range(64) if n != 7]].isnan().any()


@pytest.mark.parametrize("T", [20, 150])
def test_values_that_are_not_finite_stay_in_their_rows_of_a_large_call(T):
    from nestquant_b200 import w4
    q, s, z = make(200, 512, 64, BF16)
    w, x = w4.W4(q, s, z), torch.randn(T, 512, device="cuda").bfloat16()
    clean = w(x)
    x[T - 1, 300] = float("nan")
    x[2, 5] = float("inf")
    y = w(x)
    keep = [r for r in range(T) if r not in (2, T - 1)]
    assert torch.equal(y[keep], clean[keep]) and y[T - 1].isnan().all()
    qe, se, ze = make(200, 512, 64, BF16, E=2)             # the next expert's rows are in the same tile
    we, start = w4.W4(qe, se, ze), torch.tensor([0, T - 1, T], dtype=torch.int32, device="cuda")
    x[2, 5] = 0
    y = we(x, start=start)
    assert not y[:T - 1].isnan().any() and y[T - 1].isnan().all()


@pytest.mark.parametrize("T", [3, 16, 40])
def test_long_rows_and_few_columns_of_the_result(T):
    from nestquant_b200 import w4
    for N, K, g in ((24, 20480, 128), (7, 32768, 64), (33, 12320, 32)):
        q, s, z = make(N, K, g)
        x = torch.randn(T, K, device="cuda").half()
        check(w4.W4(q, s, z)(x, dtype=F32), x, dense(q, s, z, g), K)


def test_many_experts():
    from nestquant_b200 import w4
    E, N, K = 1024, 20, 128
    q, s, z = make(N, K, 32, E=E)
    w = w4.W4(q, s, z)
    for rows in ((torch.arange(E) % 7 == 0).int(), torch.full((E,), 2), torch.randint(0, 60, (E,), generator=torch.Generator().manual_seed(1))):
        start = torch.cat([torch.zeros(1), rows.cumsum(0)]).int().cuda()
        x = torch.randn(int(start[-1]), K, device="cuda").half()
        y = w(x, start=start, dtype=F32)
        W = dense(q, s, z, 32)
        e = torch.repeat_interleave(torch.arange(E), rows.long()).cuda()
        want = torch.einsum("pk,pnk->pn", x.double(), W[e])
        size = torch.einsum("pk,pnk->pn", x.double().abs(), W[e].abs())
        assert ((y.double() - want).abs() <= 40 * 2.0 ** -23 * size + 2.0 ** -24 * want.abs()).all()


def test_a_start_that_falls_gives_zeros_and_says_so():
    from nestquant_b200 import w4
    for T in (9, 200):
        q, s, z = make(48, 256, 64, E=4)
        w, x = w4.W4(q, s, z), torch.randn(T, 256, device="cuda").half()
        good = torch.tensor([0, 2, 5, 5, T], dtype=torch.int32, device="cuda")
        y = w(x, start=good)
        assert w.status() == 0
        for bad in ([0, 5, 2, 5, T], [0, 2, 5, -1, T], [0, 2 ** 30, 3, 4, 5]):
            assert (w(x, start=torch.tensor(bad, dtype=torch.int32, device="cuda")) == 0).all()
            assert w.status() == 2
        assert torch.equal(w(x, start=good), y)
        over = torch.tensor([0, 2, 5, 5, 2 ** 30], dtype=torch.int32, device="cuda")      # ends behind the last row
        assert torch.equal(w(x, start=over), y)


def test_large_calls_on_two_streams_at_once():
    from nestquant_b200 import w4
    q, s, z = make(640, 1024, 128)
    w, W = w4.W4(q, s, z), dense(q, s, z, 128)
    xs = [torch.randn(T, 1024, device="cuda").half() for T in (40, 300)]
    torch.cuda.synchronize()
    streams, ys = [torch.cuda.Stream() for _ in xs], []
    for _ in range(5):
        for st, x in zip(streams, xs):
            with torch.cuda.stream(st):
                ys.append((w(x), x))
    torch.cuda.synchronize()
    for y, x in ys:
        check(y, x, W, 1024)
    assert w.status() == 0


def test_the_first_calls_of_a_process_can_be_captured():
    import subprocess
    import sys
    code = """
import torch
from nestquant_b200 import routing, w4
q = torch.randint(0, 256, (64, 128), device="cuda", dtype=torch.uint8)
w = w4.W4(q, torch.full((64, 4), 0.5, device="cuda", dtype=torch.float16))
x, l = torch.ones(20, 256, device="cuda", dtype=torch.float16), torch.randn(20, 16, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    few, many = w(x[:3].clone()), w(x)
    sel, rw = routing.route(l, 4)
    o = routing.sort_picks(sel, 16)
    out = routing.combine(routing.dispatch(x, o), o, rw, dtype=torch.float32)
g.replay()
torch.cuda.synchronize()
assert torch.equal(few, many[:3]) and (out - 1).abs().max() < 4 * 2.0 ** -11, (few, out)      # weights of 16 bits that add up to 1
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_large_sums_stay_in_32_bits():
    """rows with a large common part: what is subtracted is subtracted before anything is rounded"""
    from nestquant_b200 import w4
    q, s, z = make(64, 4096, 128, zeros=True)
    x = (100 + torch.randn(4, 4096, device="cuda")).half()
    check(w4.W4(q, s, z)(x, dtype=F32), x, dense(q, s, z, 128), 4096)


def test_planes_past_32_bit_offsets():
    from nestquant_b200 import w4
    E, N, K = 180, 4096, 12288                    # 4.5 GB
    q = torch.randint(0, 256, (E, N, K // 2), device="cuda", dtype=torch.uint8)
    s = (0.01 * torch.randn(E, N, K // 128, device="cuda")).half()
    w = w4.W4(q, s)
    start = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    start[E:] = 2
    x = torch.randn(2, K, device="cuda").half()
    check(w(x, start=start), x, dense(q[-1], s[-1], None, 128), K)
    del q, w
    torch.cuda.empty_cache()


def test_captured_calls_and_other_streams():
    from nestquant_b200 import w4
    q, s, z = make(96, 512, 64)
    w, W = w4.W4(q, s, z), dense(q, s, z, 64)
    xs = [torch.randn(T, 512, device="cuda").half() for T in (1, 20)]
    for x in xs:
        w(x)
    graphs = []
    for x in xs:                                   # two graphs of one matrix, replayed side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = w(x)
        graphs.append((g, x, y))
    side = torch.cuda.Stream()
    for seed in range(3):
        for x in xs:
            x.copy_(torch.randn(x.shape, device="cuda"))
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, x, y in graphs:
            check(y, x, W, 512)


def test_a_whole_layer_of_4_bit_experts():
    """route -> sort -> dispatch -> gate | up -> SwiGLU -> down -> combine, a shared expert beside it, against 64 bits"""
    from nestquant_b200 import routing, w4
    T, E, topk, H, I = 24, 12, 3, 256, 128
    gu, dn = make(2 * I, H, 128, E=E, seed=1), make(H, I, 64, E=E, seed=2)
    sgu, sdn = make(2 * I, H, 128, seed=3), make(H, I, 64, seed=4)
    gen = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(T, H, generator=gen, device="cuda").half()
    logits = torch.randn(T, E, generator=gen, device="cuda")
    swiglu = lambda h: torch.nn.functional.silu(h[:, :I]) * h[:, I:]
    sel, rw = routing.route(logits, topk, bias=torch.zeros(E, device="cuda"), scale=2.5)
    o = routing.sort_picks(sel, E)
    h = swiglu(w4.W4(*gu)(routing.dispatch(x, o), start=o.start, dtype=F32)).half()
    out = routing.combine(w4.W4(*dn)(h, start=o.start), o, rw, dtype=F32)
    out = out + w4.W4(*sdn)(swiglu(w4.W4(*sgu)(x, dtype=F32)).half(), dtype=F32)
    G, D = dense(*gu, 128), dense(*dn, 64)
    want = swiglu(x.double() @ dense(*sgu, 128).T) @ dense(*sdn, 64).T
    p = torch.sigmoid(logits.double()).gather(1, sel)
    p = 2.5 * p / p.sum(1, keepdim=True)
    for t in range(T):
        for k in range(topk):
            e = int(sel[t, k])
            want[t] += p[t, k] * (D[e] @ swiglu((G[e] @ x[t].double())[None])[0])
    # roundings to fp16 of h, of the experts' rows and of the weights: 2^-11 of values whose sum has about this size
    assert float((out.double() - want).norm() / want.norm()) < 3 * 2.0 ** -11


def test_refusals():
    from nestquant_b200 import w4
    from nestquant_b200.capi import NestQuantError
    q, s, z = make(32, 256, 64)
    w = w4.W4(q, s, z)
    qe, se, ze = make(32, 256, 64, E=3)
    we = w4.W4(qe, se, ze)
    x = torch.zeros(4, 256, device="cuda", dtype=F16)
    start = torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in (
        lambda: w4.W4(q.int(), s), lambda: w4.W4(q, s.float()), lambda: w4.W4(q, s[:, :3]), lambda: w4.W4(q, s[:16]), lambda: w4.W4(q, s, z[:, :2]), lambda: w4.W4(q, s, z.int()),
        lambda: w4.W4(q, s[:, :1].contiguous()), lambda: w4.W4(q[:, :8].contiguous(), s[:, :1]), lambda: w4.W4(q.cpu(), s), lambda: w4.W4(q, s.cpu()), lambda: w4.W4(q[0], s[0]), lambda: w4.W4(q[:0], s[:0]),
        lambda: w(x[:, :128]), lambda: w(x.float()), lambda: w(x.cpu()), lambda: w(x[0]), lambda: w(x, dtype=BF16), lambda: w(x, start=start), lambda: we(x),
        lambda: we(x, start=start[:3]), lambda: we(x, start=start.long()), lambda: we(x, start=start.cpu()), lambda: w(x.clone().requires_grad_(True)),
    ):
        with pytest.raises(NestQuantError):
            call()
    with torch.no_grad():
        assert w(x.clone().requires_grad_(True)).shape == (4, 32)
