"""`low_rank_add`, the low-rank adapters of many requests beside a shared projection, against a restatement in 64 bits, and
the three operators of a projection run together.

Tolerances: one rounding to bf16 is 2^-8 of the value; the low-rank row and the sum over it are kept to 16 bits or more and
their sums in fp32: 2^-15 of the sum of magnitudes |scale| (|x| |a|^T) |b|^T covers 2^-16 for the low-rank row's rounding and
fp32 sums of up to 8192 and 256 terms in 32 or more parts (2^-17)."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

from ironmlx_b200 import _lib, nn, ops
from test_gpu_rows8 import bf16, check_product, check_rows, gen, mx, norm64

pytestmark = pytest.mark.gpu


def make(g, t, k, n, count, rank, scale=True):
    return dict(y=bf16(g, t, n), x=bf16(g, t, k), a=bf16(g, count, rank, k, std=k ** -0.5), b=bf16(g, count, n, rank, std=0.1),
                scale=torch.rand(count, generator=g, device="cuda") * 1.5 + 0.5 if scale else None)


def check(out, p, ids):
    y, x = p["y"].double(), p["x"].double()
    mag = torch.zeros_like(y)
    for j in range(p["a"].shape[0]):
        at = torch.nonzero(ids == j).flatten()
        s = 1.0 if p["scale"] is None else p["scale"][j].double()
        y[at] += s * (x[at] @ p["a"][j].double().T) @ p["b"][j].double().T
        mag[at] += s * (x[at].abs() @ p["a"][j].double().abs().T) @ p["b"][j].double().abs().T
    assert ((out.double() - y).abs() <= y.abs() * 2.0 ** -8 + mag * 2.0 ** -15 + 1e-38).all()
    none = (ids < 0) | (ids >= p["a"].shape[0])
    assert torch.equal(out[none], p["y"][none])


def run(p, ids, **kw):
    return ops.low_rank_add(p["y"], p["x"], p["a"], p["b"], ids, p["scale"], **kw)


@pytest.mark.parametrize("t,k,n,count,rank", [
    (1, 2048, 8192, 1, 16), (1, 8, 1, 1, 8), (2, 64, 7, 3, 8), (5, 4096, 2048, 4, 64), (16, 2048, 512, 40, 32), (48, 4096, 2048, 40, 32),
    (31, 1000, 1001, 2, 24), (64, 512, 264, 64, 256), (100, 2048, 1024, 3, 128), (130, 96, 200, 5, 16), (300, 2048, 2048, 1, 16),
    (777, 2056, 1032, 5, 40), (1100, 512, 513, 12, 64), (140, 8, 16, 1, 8), (131, 200, 72, 3, 200), (8500, 128, 200, 9, 48), (150, 64, 128, 2500, 8), (2050, 256, 384, 200, 8), (600, 4096, 136, 2, 256), (5000, 64, 96, 3, 16), (400, 1024, 2048, 2, 128), (260, 3000, 1500, 1, 256),
    (300, 512, 1030, 4, 24), (145, 64, 70, 2, 72)])
@pytest.mark.parametrize("order", ["mixed", "runs"])
def test_low_rank_add(cuda, t, k, n, count, rank, order):
    g = gen(t + k + n + rank)
    p = make(g, t, k, n, count, rank, scale=order == "mixed")
    ids = torch.randint(-1, count, (t,), generator=g, device="cuda", dtype=torch.int32)
    if order == "runs":
        ids = ids[torch.arange(t, device="cuda") // max(1, t // 7) * max(1, t // 7)].contiguous()
        ids[t - t // 9:] = -1                                           # padding
    out = run(p, ids)
    check(out, p, ids)
    assert torch.equal(out, run(p, ids))
    y = p["y"].clone()
    assert ops.low_rank_add(y, p["x"], p["a"], p["b"], ids, p["scale"], out=y) is y and torch.equal(y, out)


@pytest.mark.parametrize("t,n,count,rank", [(1, 96, 1, 16), (5, 100, 2, 8), (40, 264, 3, 64), (20, 41, 2, 128), (20, 72, 2, 200), (100, 128, 9, 256),
                                            (300, 136, 2, 16), (300, 264, 2, 64), (200, 136, 1, 128), (200, 72, 1, 256), (300, 77, 2, 24)])
def test_whole_numbers_of_24_bits_are_exact(cuda, t, n, count, rank):
    """Low-rank rows of up to 21 bits, and a y that takes the first eight bits of what is added to it: every sum is a whole
    number below 2^24, exact in fp32 in any order, so that every output is the one rounding of its sum.  (A low-rank row of 16
    bits leaves a few units of 2^19, next to outputs whose step is 8 and less.)"""
    g = gen(t + n + rank)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda")

    p = dict(x=whole(0, 65, t, 512).bfloat16(), a=whole(0, 65, count, rank, 512).bfloat16(), scale=None,
             b=((whole(0, rank, count, n, rank) < 4) * (2 * whole(0, 2, count, n, rank) - 1)).bfloat16())
    ids = whole(0, count, t).int()
    rows = torch.einsum("tk,trk->tr", p["x"].double(), p["a"].double()[ids.long()])
    add = torch.einsum("tr,tnr->tn", rows, p["b"].double()[ids.long()])
    p["y"] = -add.bfloat16()
    assert rows.max() > 2 ** 18 and torch.einsum("tr,tnr->tn", rows, p["b"].double().abs()[ids.long()]).max() < 2 ** 24
    assert torch.equal(run(p, ids), (p["y"].double() + add).float().bfloat16())


@pytest.mark.parametrize("rank,steps", [(16, 32), (64, 32), (128, 32), (256, 64)])
def test_long_sums_are_not_cut_off_too_often(cuda, rank, steps):
    """Sums of 4096 positive products, of which y takes the first eight bits.  The tensor cores cut a sum off at each addition, by
    half a unit of its last place on average, which at a share f of the whole is at most f 2^-23 of it: `steps` additions to one
    sum make it steps 2^-25 too small on average (roundings of the outputs have no such mean).  A CTA of two has 2048 of the
    values, 128 K steps, as four sums (two above a rank of 128)."""
    g = gen(rank)
    t, n = 8192, 64
    x, a = ((1 + torch.rand(*shape, generator=g, device="cuda")).bfloat16() for shape in ((t, 4096), (1, rank, 4096)))
    b = torch.zeros(1, n, rank, dtype=torch.bfloat16, device=cuda)
    b[0, torch.arange(n, device=cuda), torch.arange(n, device=cuda) % rank] = 1.0
    add = (x.double() @ a[0].double().T) @ b[0].double().T
    y = -add.bfloat16()
    out = ops.low_rank_add(y, x, a, b, torch.zeros(t, dtype=torch.int32, device=cuda))
    off = ((out.double() - (y.double() + add)) / add).mean().item()
    assert abs(off) <= steps * 2.0 ** -25, (off, steps * 2.0 ** -25)


@pytest.mark.parametrize("t,count,rank", [(129, 129, 16), (200, 150, 64), (256, 200, 16), (256, 2100, 8), (384, 300, 128), (512, 400, 16), (512, 512, 64)])
def test_more_rows_than_128_with_nearly_as_many_adapters(cuda, t, count, rank):
    """A decode batch above the size of the kernel for few rows, most of whose rows are alone with their adapter."""
    g = gen(t + count)
    p = make(g, t, 1024, 520, count, rank)
    ids = torch.randperm(count, generator=g, device="cuda")[torch.arange(t, device="cuda") % count].int()
    ids[::17] = -1
    ids[1] = ids[t - 1]
    out = run(p, ids)
    check(out, p, ids)
    assert torch.equal(out, run(p, ids))


@pytest.mark.parametrize("t", [3, 70, 700])
def test_ids_without_an_adapter(cuda, t):
    """No row has one; ids far outside; every row the last adapter.  What a row without an adapter holds is left bit for bit,
    NaN and infinities among it, whatever its x."""
    g = gen(t)
    p = make(g, t, 256, 320, 5, 16)
    p["y"][0, 5], p["y"][1, 6] = float("nan"), float("-inf")
    p["x"][0] = float("nan")
    none = torch.full((t,), -1, dtype=torch.int32, device=cuda)
    assert torch.equal(run(p, none).view(torch.int16), p["y"].view(torch.int16))
    wild = torch.tensor([-2 ** 31, 2 ** 31 - 1, 5], device=cuda).int().repeat(t)[:t].contiguous()
    assert torch.equal(run(p, wild).view(torch.int16), p["y"].view(torch.int16))
    last = torch.full((t,), 4, dtype=torch.int32, device=cuda)
    last[:2] = -1
    out = run(p, last)
    assert torch.equal(out[:2].view(torch.int16), p["y"][:2].view(torch.int16))
    check(out[2:], {**p, "y": p["y"][2:], "x": p["x"][2:]}, last[2:])


@pytest.mark.parametrize("t", [2, 40, 400])
def test_rows_that_are_not_finite_stay_alone(cuda, t):
    """A NaN or an infinity in one row's x or y, or in one adapter, changes no row beside it, also of the same adapter."""
    g = gen(t + 1)
    p = make(g, t, 512, 264, 3, 16)
    ids = (torch.arange(t, device="cuda") % 2).int()
    clean = run(p, ids)
    p["x"][1, 9] = float("nan")
    p["a"][2, 3, 4] = float("nan")                                       # an adapter of no row
    p["b"][2, 3, 4] = float("inf")
    out = run(p, ids)
    assert out[1].isnan().all()
    keep = torch.arange(t, device="cuda") != 1
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("t,n", [(3, 40), (3, 41), (200, 136), (200, 77), (1200, 264)])
@pytest.mark.parametrize("at", [1, 4])
def test_low_rank_add_at_any_place(cuda, t, n, at):
    g = gen(n)
    p = make(g, t, 128, n, 4, 16)
    ids = torch.randint(-1, 4, (t,), generator=g, device="cuda", dtype=torch.int32)
    want = run(p, ids)
    src = torch.full((t * n + 16,), 3.0, dtype=torch.bfloat16, device=cuda)
    src[at:at + t * n] = p["y"].flatten()
    buf = torch.full((t * n + 16,), 7.0, dtype=torch.bfloat16, device=cuda)
    ad = _lib.Adapters(p["a"].data_ptr(), p["b"].data_ptr(), p["scale"].data_ptr(), 4, 16)
    scratch = torch.zeros(256, dtype=torch.uint8, device=cuda)
    for dst in (buf, src):
        _lib.check(_lib.lib().imx_low_rank_add(src.data_ptr() + 2 * at, p["x"].data_ptr(), t, 128, C.byref(ad), ids.data_ptr(), n,
                                               dst.data_ptr() + 2 * at, scratch.data_ptr(), 256, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(dst[at:at + t * n].view(t, n), want)
        assert (dst[:at] == dst[0]).all() and (dst[at + t * n:] == dst[0]).all()


def test_expired_wait_gives_nan_and_a_status(cuda):
    g = gen(19)
    p = make(g, 400, 512, 520, 3, 32)
    ids = torch.randint(-1, 3, (400,), generator=g, device="cuda", dtype=torch.int32)
    want = run(p, ids)
    _lib.lib().imx_testing_low_rank_give_up(1)
    try:
        out = run(p, ids)
        torch.cuda.synchronize()
    finally:
        _lib.lib().imx_testing_low_rank_give_up(0)
    assert out[ids >= 0].isnan().all() and torch.equal(out[ids < 0], p["y"][ids < 0])
    with pytest.raises(_lib.IronMLXError):
        ops.check_status(cuda)
    assert torch.equal(run(p, ids), want)
    ops.check_status(cuda)


FIRST_CALL_IN_A_CAPTURE = """
import torch
from ironmlx_b200 import IronMLXError, _lib, ops
t, k, n = 300, 512, 512
y, x, ids = torch.zeros(t, n, device="cuda").bfloat16(), torch.ones(t, k, device="cuda").bfloat16(), torch.zeros(t, dtype=torch.int32, device="cuda")
a, b = torch.ones(1, 16, k, device="cuda").bfloat16(), torch.ones(1, n, 16, device="cuda").bfloat16()
packed, scales = torch.full((t, k // 4), 0x38383838, dtype=torch.int32, device="cuda"), torch.full((t, k // 32), 127, dtype=torch.uint8, device="cuda")
hooks = dict(adapters=_lib.lib().imx_testing_low_rank_give_up, product=_lib.lib().imx_testing_mxfp8_give_up)
calls = dict(adapters=lambda: ops.low_rank_add(y, x, a, b, ids), product=lambda: ops.mxfp8_matmul((packed, scales), packed, scales))
values = dict(adapters=16.0 * k, product=float(k))
for which in (FIRST, "adapters", "product"):
    for give_up in (1, 0):
        hooks[which](give_up)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, after = calls[which](), torch.ones(4096, device="cuda")
        hooks[which](0)
        for _ in range(2):
            graph.replay()
            graph.replay()
            torch.cuda.synchronize()
            assert (after == 1).all()
            if give_up:
                assert out.isnan().all()
                try:
                    ops.check_status()
                    raise SystemExit("not reported")
                except IronMLXError as e:
                    assert e.code == _lib.ERR_DEVICE
            else:
                assert (out == values[which]).all()
            ops.check_status()
"""


@pytest.mark.parametrize("first", ["adapters", "product"])
def test_first_call_in_a_capture_reports_its_replays(cuda, first):
    """In a process of its own, whose first call of the operators is captured: every replay whose waits run out is reported."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE.replace("FIRST", repr(first))], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.parametrize("rank", [16, 64, 128, 256])
@pytest.mark.parametrize("cta", [0, 1, 7])
def test_one_cta_of_a_cluster_gives_up(cuda, rank, cta):
    """A CTA that gives up in the first product has a part of its rows' sums that all CTAs of its cluster need: no output of
    theirs is a number, the status is reported once, the next call is right again."""
    g = gen(24)
    p = make(g, 400, 512, 1040, 3, rank)
    ids = torch.randint(-1, 3, (400,), generator=g, device="cuda", dtype=torch.int32)
    want = run(p, ids)
    _lib.lib().imx_testing_low_rank_give_up(2 + cta)
    try:
        out = run(p, ids)
        torch.cuda.synchronize()
    finally:
        _lib.lib().imx_testing_low_rank_give_up(0)
    assert out[ids >= 0].isnan().all() and torch.equal(out[ids < 0], p["y"][ids < 0])
    with pytest.raises(_lib.IronMLXError):
        ops.check_status(cuda)
    ops.check_status(cuda)
    assert torch.equal(run(p, ids), want)


def test_as_many_rows_as_an_int_counts(cuda):
    """2^31 - 1 rows: the last block of 8192 ends where 31 bits end.  Few rows have an adapter, all others stay as they are."""
    rows = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("64 GB of memory needed")
    g = gen(23)
    p = make(g, 1, 8, 1, 2, 8)
    x, y = torch.empty(rows, 8, dtype=torch.bfloat16, device=cuda), torch.full((rows, 1), 3.0, dtype=torch.bfloat16, device=cuda)
    ids = torch.full((rows,), -1, dtype=torch.int32, device=cuda)
    at = [0, 8191, 8192, 2 ** 30, rows - 8192, rows - 8191, rows - 2, rows - 1]
    small = {**p, "x": bf16(g, 8, 8), "y": y[:8].clone()}
    for i, row in enumerate(at):
        x[row], ids[row] = small["x"][i], i % 2
    run({**p, "x": x, "y": y}, ids, out=y)
    check(torch.stack([y[row] for row in at]), small, torch.stack([ids[row] for row in at]))
    for row in at:
        y[row] = 3.0
    assert all((part == 3).all() for part in y.split(1 << 28))


def test_adapters_on_streams(cuda):
    g = gen(20)
    p, q = make(g, 300, 512, 512, 6, 16), make(g, 24, 512, 512, 6, 16)
    ip, iq = (torch.randint(-1, 6, (t,), generator=g, device="cuda", dtype=torch.int32) for t in (300, 24))
    want = run(p, ip), run(q, iq)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [run((p, q)[i % 2], (ip, iq)[i % 2], stream=streams[i // 2 % 2]) for i in range(24)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))
    assert ops.low_rank_add(p["y"][:0], p["x"][:0], p["a"], p["b"], ip[:0]).shape == (0, 512)


def test_adapters_beside_products(cuda):
    """Tiles of adapters (two CTAs an SM, 128 columns of tensor memory each) and pairs of the product (all 512) on two streams at
    the same time: the values of the calls alone."""
    g = gen(77)
    p = make(g, 700, 1024, 2048, 5, 16)
    ids = torch.randint(-1, 5, (700,), generator=g, device="cuda", dtype=torch.int32)
    rows = ops.quantize(torch.randn(700, 2048, generator=g, device="cuda"), mode="mxfp8")[:2]
    w = ops.quantize(torch.randn(1024, 2048, generator=g, device="cuda"), mode="mxfp8")[:2]
    alone = run(p, ids), ops.mxfp8_matmul(rows, *w)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [(run(p, ids, stream=streams[i & 1]), ops.mxfp8_matmul(rows, *w, stream=streams[1 - (i & 1)])) for i in range(40)]
    torch.cuda.synchronize()
    ops.check_status()
    assert all(torch.equal(x, alone[0]) and torch.equal(y, alone[1]) for x, y in got)


@pytest.mark.parametrize("rank", [16, 64, 136, 256])
def test_adapters_beside_pairs_with_two_term_weights(cuda, rank):
    """Tiles of adapters and the pairs of CTAs of a 6-bit projection (which hold all of tensor memory and need little shared
    memory) on streams of their own at the same time, and tiles of a small rank beside both: the values of the calls alone."""
    g = gen(78)
    p, q = make(g, 700, 1024, 2048, 5, rank), make(g, 600, 512, 1024, 3, 8)
    ip, iq = (torch.randint(-1, 3, (t,), generator=g, device="cuda", dtype=torch.int32) for t in (700, 600))
    w = nn.QuantizedLinear.new(*ops.quantize(torch.randn(2048, 1024, generator=g, device="cuda") * 0.05, bits=6, group_size=64), 64, 6)
    x = bf16(g, 1500, 1024)
    alone = run(p, ip), run(q, iq), w.forward_with_stream(x)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()

    def project():
        with torch.cuda.stream(streams[2]):
            return w.forward_with_stream(x)

    got = [(run(p, ip, stream=streams[i % 2]), run(q, iq, stream=streams[1 - i % 2]), project()) for i in range(40)]
    torch.cuda.synchronize()
    ops.check_status()
    assert all(torch.equal(a, b) for three in got for a, b in zip(three, alone))


@pytest.mark.parametrize("kind", ["dense", "affine", "mxfp8"])
def test_projection_with_adapters(cuda, kind):
    g = gen(21)
    p = make(g, 30, 512, 256, 3, 16)
    w = torch.randn(256, 512, generator=g, device="cuda") * 0.05
    layer = nn.Linear(w.bfloat16()) if kind == "dense" else (
        nn.QuantizedLinear.new(*ops.quantize(w), 64, 4) if kind == "affine" else
        nn.QuantizedLinear.new_with_mode(*ops.quantize(w, mode="mxfp8"), 32, 8, "mxfp8"))
    ids = torch.randint(-1, 3, (30,), generator=g, device="cuda", dtype=torch.int32)
    out = layer.forward_with_adapters(p["x"], nn.LowRankAdapters(p["a"], p["b"], p["scale"]), ids)
    check(out, {**p, "y": layer.forward_with_stream(p["x"])}, ids)


@pytest.mark.parametrize("t", [1, 24, 200])
def test_norm_product_and_adapters_together(cuda, t):
    """The three as a decoder layer runs them -- residual and norm, the projection of the 8-bit rows, the adapters of the bf16
    rows -- eagerly, then captured and replayed with other inputs in the same buffers while another captured run of its own
    is replayed on another stream."""
    g = gen(22)
    hidden, n = 512, 768
    norm = nn.RMSNorm.new(bf16(g, hidden, std=0.1) + 1, 1e-6)
    layer = nn.QuantizedLinear.new_with_mode(*mx(g, n, hidden, 0.02), None, 32, 8, "mxfp8")
    p = make(g, t, hidden, n, 4, 16)
    adapters = nn.LowRankAdapters(p["a"], p["b"], p["scale"])

    def inputs():
        return [bf16(g, t, hidden), bf16(g, t, hidden, std=2.0), torch.randint(-1, 4, (t,), generator=g, device="cuda", dtype=torch.int32)]

    def step(x, r, ids):
        h, y, rows = norm.forward_residual(x, r, "both")
        base = layer.forward_rows(rows)
        return h, y, rows.packed, rows.scales, base, adapters.add(base, y, ids)

    first = inputs()
    h, y, packed, scales, base, out = step(*first)
    v, u = norm64(first[0], first[1], norm.weight)
    check_rows((packed, scales), u)
    check_product(base, (packed, scales), (layer.weight, layer.scales))
    check(out, {**p, "y": base, "x": y}, first[2])

    graphs, bufs, outs = [], [], []
    for _ in range(2):
        buf = [b.clone() for b in first]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(*buf)
        graphs.append((graph, side))
        bufs.append(buf)
        outs.append(got)
    torch.cuda.synchronize()
    for _ in range(3):
        fresh = [inputs(), inputs()]
        for buf, new in zip(bufs, fresh):
            for b, v in zip(buf, new):
                b.copy_(v)
        torch.cuda.synchronize()
        for graph, side in graphs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for got, new in zip(outs, fresh):
            assert all(torch.equal(a, b) for a, b in zip(got, step(*new)))
