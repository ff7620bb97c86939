"""`add_rms_norm` (residual + RMSNorm + 8-bit rows) and `mxfp8_matmul` (8-bit rows times an mxfp8 weight) against plain
restatements in 64 bits.

Tolerances: rounding to bf16 is off by at most 2^-8 of the value, to e4m3 by at most 2^-4 (2^-10 of the scale below its
smallest normal number).  The norm's factor carries fp32 sums of at most 32768 / 512 + 20 additions and one rsqrtf (2^-22):
under 2^-16 in all.  A product's fp32 sum adds in / 32 blocks; each addition, and the 32 products within, are taken to be off
by at most 2^-22 of the sum of magnitudes."""
import ctypes as C

import numpy as np
import pytest
import torch

from ironmlx_b200 import _lib, nn, ops
from oracle import formats as F
from oracle import moe as O

pytestmark = pytest.mark.gpu
EPS = 1e-6


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def bf16(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).bfloat16()


def values(packed, scales):
    """The numbers of mxfp8 rows, in 64 bits."""
    q = packed.contiguous().view(torch.float8_e4m3fn).double()
    return (q.unflatten(-1, (-1, 32)) * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)


def norm64(x, residual, weight):
    v = x.double() + (0 if residual is None else residual.double())
    u = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v, u if weight is None else u * weight.double()


def check_rows(rows, u):
    """Codes and scales are a rounding of u by imx_quantize's rule."""
    packed, scales = rows
    e = scales.double() - 127
    amax = u.abs().unflatten(-1, (-1, 32)).amax(-1)
    tiny = amax <= 448 * 2.0 ** -127
    assert (e[tiny] == -127).all()
    hi, lo = 448 * torch.exp2(e), 224 * torch.exp2(e)
    assert (amax <= hi * (1 + 2.0 ** -15))[~tiny].all() and (amax > lo * (1 - 2.0 ** -15))[~tiny].all()
    half_step = torch.maximum(u.abs() * 2.0 ** -4, (2.0 ** -10 * torch.exp2(e)).repeat_interleave(32, -1))
    assert ((values(packed, scales) - u).abs() <= half_step * (1 + 2.0 ** -12) + u.abs() * 2.0 ** -15).all()


@pytest.mark.parametrize("rows,hidden", [(1, 32), (1, 2048), (2, 40), (3, 8), (7, 96), (64, 2048), (129, 5120), (2000, 160),
                                         (5, 16384), (3, 32768), (1500, 2048), (333, 8192), (700, 1056)])
@pytest.mark.parametrize("residual,weight,out", [(True, True, "both"), (True, False, "mxfp8"), (False, True, "bf16")])
def test_add_rms_norm(cuda, rows, hidden, residual, weight, out):
    if hidden % 32:
        out = "bf16"
    g = gen(rows + hidden)
    x = bf16(g, rows, hidden) * torch.where(torch.rand(hidden, generator=g, device="cuda") < 0.02, 30.0, 1.0).bfloat16()
    x[rows // 2] *= 1e-4
    r = bf16(g, rows, hidden, std=2.0) if residual else None
    w = (bf16(g, hidden, std=0.2) + 1) if weight else None
    h, y, rows8 = ops.add_rms_norm(x, r, w, EPS, out)
    if residual:
        assert torch.equal(h, (x.float() + r.float()).bfloat16())
    else:
        assert h is x
    v, u = norm64(x, r, w)
    assert (y is None) == (out == "mxfp8") and (rows8 is None) == (out == "bf16")
    if y is not None:
        assert ((y.double() - u).abs() <= u.abs() * (2.0 ** -8 + 2.0 ** -15) + 1e-38).all()
    if rows8 is not None:
        check_rows(rows8, u)
    again = ops.add_rms_norm(x, r, w, EPS, out)
    for a, b in zip((h, y) + tuple(rows8 or ()), again[:2] + tuple(again[2] or ())):
        assert (a is None and b is None) or torch.equal(a, b)


def test_rows_are_those_of_quantize_where_the_factor_is_one(cuda):
    """Rows of +-1 have the factor rsqrt(1) = 1 exactly, so that u is the weight: bit for bit quantize's codes and scales, over
    a range of magnitudes, with zeros, amax at 448 times a power of two and next to it."""
    g = gen(3)
    w = (torch.randn(4096, generator=g, device="cuda") * torch.exp2(torch.randint(-60, 60, (128,), generator=g, device="cuda").float()).repeat_interleave(32)).bfloat16()
    w[:32] = 0
    w[32:64] = 448.0
    w[64:96], w[64] = 1.0, 450.0
    w[96:128], w[97] = 0.001, -14.0
    w[128:160] = 2.0 ** -126
    x = torch.where(torch.rand(5, 4096, generator=g, device="cuda") < 0.5, -1.0, 1.0).bfloat16()
    _, y, rows = ops.add_rms_norm(x, None, w, 0.0, "both")
    u = x.float() * w.float()
    assert torch.equal(y.float(), u)
    packed, scales, _ = ops.quantize(u, mode="mxfp8")
    assert torch.equal(rows.scales, scales) and torch.equal(rows.packed, packed)
    p, s = F.mxfp8_quantize(u.cpu().numpy())
    assert np.array_equal(rows.packed.cpu().numpy().view(np.uint32), p) and np.array_equal(rows.scales.cpu().numpy(), s)


@pytest.mark.parametrize("rows,hidden", [(2048, 8192), (4096, 512)])
def test_codes_next_to_the_middle_of_two(cuda, rows, hidden):
    """Where the sum of squares is exact the codes are those of the formula in 64 bits, all of them: fp32's roundings alone put
    some of 17 million on the other side of the middle between two codes."""
    g = gen(rows)
    x = torch.where(torch.rand(rows, hidden, generator=g, device="cuda") < torch.rand(rows, 1, generator=g, device="cuda"), 2.0, -1.0).bfloat16()
    w = (1 + torch.randn(hidden, generator=g, device="cuda").abs()).bfloat16()
    _, _, got = ops.add_rms_norm(x, None, w, 0.0, "mxfp8")
    v = x.double()
    u = v / torch.sqrt((v * v).mean(-1, keepdim=True)) * w.double()
    scaled = u / torch.exp2(got.scales.double() - 127).repeat_interleave(32, -1)
    step = torch.exp2(torch.floor(torch.log2(scaled.abs())) - 3)         # (no value is below the smallest normal number)
    want = (torch.round(scaled / step) * step).clamp(-448, 448)
    assert (scaled.abs() > 2.0 ** -6).all() and torch.equal(got.packed.view(torch.float8_e4m3fn).double(), want)


@pytest.mark.parametrize("rows,hidden", [(8192, 2048), (8192, 1024), (2048, 8192), (512, 32768)])
def test_codes_of_normal_rows(cuda, rows, hidden):
    """Rows with a residual, whose sums of squares fp32 rounds: v in fp32, all that follows in 64 bits, and all codes above the
    smallest normal number are the formula's."""
    g = gen(rows + hidden)
    x, r, w = bf16(g, rows, hidden, std=0.5), bf16(g, rows, hidden, std=2.0), bf16(g, hidden, std=0.1) + 1
    _, _, got = ops.add_rms_norm(x, r, w, EPS, "mxfp8")
    v = (x.float() + r.float()).double()
    u = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w.double()
    scaled = u / torch.exp2(got.scales.double() - 127).repeat_interleave(32, -1)
    step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))) - 3)
    want = (torch.round(scaled / step) * step).clamp(-448, 448)
    normal = scaled.abs() > 2.0 ** -6
    assert torch.equal(got.packed.view(torch.float8_e4m3fn).double()[normal], want[normal])


@pytest.mark.parametrize("rows,hidden", [(2048, 8192), (4096, 2048)])
@pytest.mark.parametrize("residual", [False, True])
def test_small_codes_next_to_the_middle_of_two(cuda, rows, hidden, residual):
    """A large value in every 32, so that the others are below the smallest normal number of e4m3 or around it, where codes are
    steps of 2^-9 of the scale: they are the formula's, all of them.  (Rows of 2 and -1 whose mean square is a square, 2401 / 1024,
    have values on the middle itself, which 64 bits miss by 2^-52.  Nothing else is nearer than 2^-48 to it there: a value in
    steps is the root of v^2 w^2 hidden 2^c / M with whole M <= 2^15 and an 8-bit w, the middle's square a quarter of a whole
    number, so that they are equal or 2^-30 apart.)"""
    g = gen(rows + residual)
    if residual:
        x, r = bf16(g, rows, hidden, std=0.5), bf16(g, rows, hidden, std=2.0)
    else:
        x, r = torch.where(torch.rand(rows, hidden, generator=g, device="cuda") < torch.rand(rows, 1, generator=g, device="cuda"), 2.0, -1.0).bfloat16(), None
    w = torch.exp2(-16 + 3 * torch.rand(hidden, generator=g, device="cuda")).bfloat16()
    w[::32] = 1.0
    _, _, got = ops.add_rms_norm(x, r, w, 0.0, "mxfp8")
    v = (x.float() + r.float()).double() if residual else x.double()
    u = v / torch.sqrt((v * v).mean(-1, keepdim=True)) * w.double()
    scaled = u / torch.exp2(got.scales.double() - 127).repeat_interleave(32, -1)
    step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))) - 3)
    steps = scaled / step
    middle = torch.floor(steps) + 0.5
    steps = torch.where((steps - middle).abs() < 2.0 ** -48, middle, steps)
    want = (torch.round(steps) * step).clamp(-448, 448)
    assert (scaled.abs() < 2.0 ** -6).double().mean() > 0.5 and torch.equal(got.packed.view(torch.float8_e4m3fn).double(), want)


def four_squares(n, most):
    """Whole numbers of at most `most` whose squares add up to n."""
    for a in range(min(most, int(n ** 0.5)), -1, -1):
        for b in range(min(a, int((n - a * a) ** 0.5)), -1, -1):
            left = n - a * a - b * b
            for c in range(min(b, int(left ** 0.5)), -1, -1):
                d = round((left - c * c) ** 0.5)
                if d <= c and d * d == left - c * c:
                    return a, b, c, d
    return None


def test_scales_next_to_their_border(cuda):
    """Rows of whole numbers whose largest, 7 m, has the squares' sum 2^14 m^2 + d: the norm of the largest is 7 m sqrt(4096 / sum),
    for d = 0 exactly 3.5 = 448 * 2^-7, the largest value of the scale 2^-7; a d of one is 2^-25 of it.  The scale is the
    formula's, which whole numbers tell: 2^-7 for d >= 0, 2^-6 for d < 0."""
    r = np.random.default_rng(5)
    rows, want = [], []
    for m in range(20, 37):
        for d in (-3, -1, 0, 0, 1, 2):
            v = r.integers(-int(3.4 * m), int(3.4 * m) + 1, 4096)
            v[0], v[5:9] = 7 * m * (1 if d % 2 else -1), 0
            total, i = 2 ** 14 * m * m + d, 4095
            while not 0 <= total - int((v * v).sum()) <= 90 * m * m:                       # (four squares below 6 m hold it)
                v[i], i = (0 if (v * v).sum() > total else 5 * m), i - 1
            v[5:9] = four_squares(total - int((v * v).sum()), 7 * m - 1)
            assert (v * v).sum() == total and i > 64 and (abs(v[1:]) < 7 * m).all()
            rows.append(v)
            want.append(120 if d >= 0 else 121)
    x = torch.tensor(np.array(rows), device=cuda).bfloat16()
    assert (x.cpu().double().numpy() == np.array(rows)).all()
    _, _, got = ops.add_rms_norm(x, None, None, 0.0, "mxfp8")
    assert got.scales[:, 0].tolist() == want
    _, _, got = ops.add_rms_norm(x * 0.5, (x * 0.5), None, 0.0, "both")                    # the same sum, from two halves
    assert got.scales[:, 0].tolist() == want
    u = x.double() / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True))
    check_rows(got, u)


def test_norm_in_place_and_leading_dimensions(cuda):
    g = gen(4)
    x, r, w = bf16(g, 2, 37, 1056), bf16(g, 2, 37, 1056), bf16(g, 1056)
    h, y, rows = ops.add_rms_norm(x, r, w, EPS, "both")
    assert h.shape == y.shape == x.shape and rows.packed.shape == (2, 37, 264) and rows.scales.shape == (2, 37, 33)
    lib, s = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for into_x in (True, False):                 # h over x and y over the residual, and the other way round
        a, b = x.clone(), r.clone()
        ph, py = (a, b) if into_x else (b, a)
        _lib.check(lib.imx_add_rms_norm(a.data_ptr(), b.data_ptr(), 74, 1056, w.data_ptr(), EPS, ph.data_ptr(), py.data_ptr(), None, None, s))
        assert torch.equal(ph, h) and torch.equal(py, y)


def test_norm_writes_its_rows_only(cuda):
    g = gen(5)
    x, w = bf16(g, 9, 96), bf16(g, 96)
    lib, s = _lib.lib(), torch.cuda.current_stream().cuda_stream
    buf = {k: torch.full((n,), 0x5a, dtype=torch.uint8, device=cuda) for k, n in dict(h=4096, y=4096, q=4096, s=512).items()}
    _lib.check(lib.imx_add_rms_norm(x.data_ptr(), x.data_ptr(), 9, 96, w.data_ptr(), EPS, buf["h"][512:].data_ptr(), buf["y"][512:].data_ptr(),
                                    buf["q"][512:].data_ptr(), buf["s"][65:].data_ptr(), s))
    for k, at, n in (("h", 512, 9 * 192), ("y", 512, 9 * 192), ("q", 512, 9 * 96), ("s", 65, 27)):
        assert (buf[k][:at] == 0x5a).all() and (buf[k][at + n:] == 0x5a).all(), k
    _, y, rows = ops.add_rms_norm(x, x, w, EPS, "both")
    assert torch.equal(buf["y"][512:512 + 9 * 192].view(torch.bfloat16).view(9, 96), y)
    assert torch.equal(buf["s"][65:92].view(9, 3), rows.scales)


def test_norm_of_as_many_rows_as_an_int_counts(cuda):
    """2^31 - 1 rows of eight, in place: rows of ones stay ones (the factor of 1e-6 is lost in bf16), those at the ends and around
    the middle are the norms of what was there."""
    rows = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("48 GB of memory needed")
    g = gen(7)
    x = torch.ones(rows, 8, dtype=torch.bfloat16, device=cuda)
    at, few = [0, 1, 2 ** 30, rows - 9, rows - 8, rows - 7, rows - 2, rows - 1], bf16(g, 8, 8)
    for i, row in enumerate(at):
        x[row] = few[i]
    want = ops.add_rms_norm(few, None, None, EPS)[1]
    _lib.check(_lib.lib().imx_add_rms_norm(x.data_ptr(), None, rows, 8, None, EPS, None, x.data_ptr(), None, None,
                                           torch.cuda.current_stream().cuda_stream))
    assert torch.equal(torch.stack([x[row] for row in at]), want)
    for row in at:
        x[row] = 1.0
    assert all((part == 1).all() for part in x.split(1 << 26))


def test_norm_of_infinities_and_nan(cuda):
    """What is not finite stays in its row: a NaN makes the row NaN, an infinity its own place NaN and the rest zero (its
    factor is zero), in bf16 and in 8 bits alike."""
    g = gen(6)
    x = bf16(g, 4, 512)
    clean = ops.add_rms_norm(x, None, None, EPS, "both")
    x[1, 100], x[2, 33] = float("nan"), float("-inf")
    _, y, rows = ops.add_rms_norm(x, None, None, EPS, "both")
    v = values(rows.packed, rows.scales)
    assert y[1].isnan().all() and v[1].isnan().all()
    assert y[2, 33].isnan() and v[2, 33].isnan() and y[2].isnan().sum() == 1 and v[2].isnan().sum() == 1
    assert (y[2].nan_to_num(0) == 0).all()
    for i in (0, 3):
        assert torch.equal(y[i], clean[1][i]) and torch.equal(rows.packed[i], clean[2].packed[i])


# ── products of 8-bit rows ──────────────────────────────────────────────────
def mx(g, rows, n, std=1.0):
    return ops.quantize(torch.randn(rows, n, generator=g, device="cuda") * std, mode="mxfp8")[:2]


def check_product(y, rows, w):
    a, b = values(*rows), values(*w)
    ref, mag = a @ b.T, a.abs() @ b.abs().T
    bound = ref.abs() * 2.0 ** -8 + mag * (a.shape[1] // 32 * 2.0 ** -22) + 1e-38
    assert ((y.double() - ref).abs() <= bound).all()
    if y.numel() > 1000:
        assert O.rel_l2(y.float().cpu().numpy(), ref.cpu().numpy()) <= 2e-3


@pytest.mark.parametrize("m,n_in,n_out", [
    (1, 32, 1), (1, 2048, 8192), (1, 544, 129), (2, 64, 7), (5, 96, 40), (8, 4096, 512), (16, 512, 1000), (17, 160, 128), (33, 2048, 384),
    (64, 2048, 2048), (65, 128, 256), (100, 8192, 64), (128, 1056, 136), (129, 2048, 1024), (200, 512, 4096), (300, 4128, 520),
    (777, 4096, 2048), (1000, 64, 2000), (1025, 2048, 2056), (2300, 512, 777), (513, 96, 8200), (4100, 1024, 1280),
    (400, 2080, 2501), (390, 2112, 2504), (5, 512, 20000), (40, 1056, 19001), (20, 256, 40010)])
def test_mxfp8_matmul(cuda, m, n_in, n_out):
    g = gen(m + n_in + n_out)
    rows, w = mx(g, m, n_in), mx(g, n_out, n_in, 0.02)
    y = ops.mxfp8_matmul(rows, *w)
    assert y.shape == (m, n_out) and y.dtype == torch.bfloat16
    check_product(y, rows, w)
    assert torch.equal(y, ops.mxfp8_matmul(rows, *w))
    ops.check_status(cuda)


@pytest.mark.parametrize("m,n_in,n_out", [(3, 512, 200), (48, 2048, 256), (130, 1152, 300), (700, 256, 1030), (390, 2112, 2504), (8, 544, 20004)])
def test_mxfp8_matmul_of_whole_numbers_is_exact(cuda, m, n_in, n_out):
    """Codes -1, 0, 1 with scales 2^-2 .. 2^2 (a different one for every block): sums are multiples of 2^-4 under 2^16, exact
    in fp32 in any order, so that every output is the one rounding of its sum.  A scale that reaches the wrong row, column or
    block shows."""
    g = gen(9)

    def exact(r):
        q = torch.randint(-1, 2, (r, n_in), generator=g, device="cuda").float().to(torch.float8_e4m3fn)
        return q.view(torch.int32), torch.randint(125, 130, (r, n_in // 32), generator=g, device="cuda").to(torch.uint8)

    rows, w = exact(m), exact(n_out)
    assert torch.equal(ops.mxfp8_matmul(rows, *w), (values(*rows) @ values(*w).T).float().bfloat16())


@pytest.mark.parametrize("m,n_in,n_out,y_at,s_at", [(5, 512, 200, 1, 1), (40, 2048, 264, 4, 4), (140, 640, 136, 2, 3), (300, 512, 512, 3, 2),
                                                    (1100, 544, 1024, 8, 16), (400, 2080, 2504, 8, 1)])
def test_mxfp8_matmul_at_any_place(cuda, m, n_in, n_out, y_at, s_at):
    """y at any bf16 value, scales at any byte: the values of the aligned call, nothing around them is written."""
    g = gen(10)
    rows, w = mx(g, m, n_in), mx(g, n_out, n_in, 0.02)
    want = ops.mxfp8_matmul(rows, *w)
    buf = torch.full((m * n_out + 32,), 7.0, dtype=torch.bfloat16, device=cuda)

    def moved(s):
        b = torch.full((s.numel() + 64,), 255, dtype=torch.uint8, device=cuda)       # NaN scales around
        b[s_at:s_at + s.numel()] = s.flatten()
        return b

    xs, ws = moved(rows[1]), moved(w[1])
    qt = _lib.QTensor(w[0].data_ptr(), ws.data_ptr() + s_at, None, 1.0)
    scratch = torch.zeros(256, dtype=torch.uint8, device=cuda)
    _lib.check(_lib.lib().imx_mxfp8_matmul(rows[0].data_ptr(), xs.data_ptr() + s_at, m, C.byref(qt), n_out, n_in, buf.data_ptr() + 2 * y_at,
                                           scratch.data_ptr(), 256, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(buf[y_at:y_at + m * n_out].view(m, n_out), want)
    assert (buf[:y_at] == 7).all() and (buf[y_at + m * n_out:] == 7).all()
    assert (scratch == 0).all()


@pytest.mark.parametrize("m,n_out", [(4, 300), (300, 520)])
def test_mxfp8_matmul_of_nan(cuda, m, n_out):
    """A NaN code or scale reaches its row's (its column's) outputs and no others; the extreme scales are powers of two too."""
    g = gen(11)
    rows, w = mx(g, m, 512), mx(g, n_out, 512)
    clean = ops.mxfp8_matmul(rows, *w)
    rows[0].view(torch.uint8)[1, 77] = 0x7f
    w[1][7, 3] = 255
    y = ops.mxfp8_matmul(rows, *w)
    assert y[1].isnan().all() and y[:, 7].isnan().all()
    keep = torch.ones(m, n_out, dtype=torch.bool, device=cuda)
    keep[1], keep[:, 7] = False, False
    assert torch.equal(y[keep], clean[keep])
    rows, w = mx(g, m, 512), mx(g, n_out, 512)
    rows[1].fill_(254)
    w[1].fill_(0)                                 # 2^127 * 2^-127
    check_product(ops.mxfp8_matmul(rows, *w), (rows[0], torch.full_like(rows[1], 127)), (w[0], torch.full_like(w[1], 127)))


def test_products_on_two_streams_and_other_shapes(cuda):
    """Calls of two streams at the same time, leading dimensions, slices of larger tensors, an empty batch."""
    g = gen(12)
    rows, w = mx(g, 96, 2048), mx(g, 1024, 2048, 0.02)
    want = ops.mxfp8_matmul(rows, *w)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [ops.mxfp8_matmul(rows, *w, stream=streams[i & 1]) for i in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    three = ops.mxfp8_matmul((rows[0].view(4, 24, 512), rows[1].view(4, 24, 64)), *w)
    assert torch.equal(three.view(96, 1024), want)
    assert torch.equal(ops.mxfp8_matmul((rows[0][5:20], rows[1][5:20]), w[0][128:640], w[1][128:640]), want[5:20, 128:640])
    assert ops.mxfp8_matmul((rows[0][:0], rows[1][:0]), *w).shape == (0, 1024)


def test_layers(cuda):
    """`RMSNorm.forward_residual` into `QuantizedLinear.forward_rows`, and that an affine weight is refused."""
    g = gen(13)
    x, r, wn = bf16(g, 70, 512), bf16(g, 70, 512), bf16(g, 512, std=0.1) + 1
    w = mx(g, 256, 512, 0.02)
    h, y, rows = nn.RMSNorm.new(wn, EPS).forward_residual(x, r, "both")
    layer = nn.QuantizedLinear.new_with_mode(w[0], w[1], None, 32, 8, "mxfp8")
    out = layer.forward_rows(rows)
    check_product(out, rows, w)
    # next to the same layer on bf16 rows: what 8 bits cost (each value 2^-4 at the most, 2.6e-2 on average)
    assert O.rel_l2(out.float().cpu().numpy(), layer.forward_with_stream(y).float().cpu().numpy()) <= 2.0 ** -4
    q4 = ops.quantize(torch.randn(256, 512, generator=g, device="cuda"))
    with pytest.raises(_lib.IronMLXError):
        nn.QuantizedLinear.new(*q4, 64, 4).forward_rows(rows)


@pytest.mark.parametrize("m,n_in,n_out", [(8, 2048, 256), (600, 512, 1024), (128, 64, 40000), (400, 2080, 2504), (8, 256, 20000)])
def test_expired_wait_gives_nan_and_a_status(cuda, m, n_in, n_out):
    """With every wait giving up at once nothing is copied or multiplied: outputs are NaN, the status is reported once, the
    next call is right again."""
    g = gen(14)
    rows, w = mx(g, m, n_in), mx(g, n_out, n_in, 0.02)
    want = ops.mxfp8_matmul(rows, *w)
    ops.check_status(cuda)
    _lib.lib().imx_testing_mxfp8_give_up(1)
    try:
        y = ops.mxfp8_matmul(rows, *w)
        torch.cuda.synchronize()
    finally:
        _lib.lib().imx_testing_mxfp8_give_up(0)
    assert y.isnan().all()
    with pytest.raises(_lib.IronMLXError) as e:
        ops.check_status(cuda)
    assert e.value.code == _lib.ERR_DEVICE
    ops.check_status(cuda)
    assert torch.equal(ops.mxfp8_matmul(rows, *w), want)


@pytest.mark.parametrize("m,n_in,n_out", [(1, 2048, 512), (8, 2048, 256), (20, 4096, 300), (64, 4096, 512)])
@pytest.mark.parametrize("rank", [0, 1])
def test_one_cta_of_a_cut_reduction_gives_up(cuda, m, n_in, n_out, rank):
    """Where a cluster cuts the reduction and one CTA of it gives up, no output of the cluster has all its parts: all are NaN,
    the status is reported once, the next call is right again."""
    g = gen(15)
    rows, w = mx(g, m, n_in), mx(g, n_out, n_in, 0.02)
    want = ops.mxfp8_matmul(rows, *w)
    for _ in range(5):
        _lib.lib().imx_testing_mxfp8_give_up(2 + rank)
        try:
            y = ops.mxfp8_matmul(rows, *w)
            torch.cuda.synchronize()
        finally:
            _lib.lib().imx_testing_mxfp8_give_up(0)
        assert y.isnan().all()
        with pytest.raises(_lib.IronMLXError):
            ops.check_status(cuda)
        ops.check_status(cuda)
        assert torch.equal(ops.mxfp8_matmul(rows, *w), want)
