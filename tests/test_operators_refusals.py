"""What `imx_add_rms_norm`, `imx_mxfp8_matmul` and `imx_low_rank_add` refuse, and that they refuse it on the host: the
addresses given here are not memory, no GPU is needed."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

from ironmlx_b200 import _lib, nn, ops

A, B, D, E, F, G = (0x100000000 * i for i in range(1, 7))       # far apart, aligned


def refused(status, needle, code=_lib.ERR_INVALID):
    assert status == code and needle in _lib.lib().imx_last_error(), _lib.lib().imx_last_error()


def norm(x=A, residual=B, n=4, hidden=64, w=D, h=E, y=F, q=G, s=G + 0x1000):
    return _lib.lib().imx_add_rms_norm(x, residual, n, hidden, w, 1e-6, h, y, q, s, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(n=-1), b"negative"), (dict(hidden=0), b"row length"), (dict(hidden=12), b"row length"), (dict(hidden=32776), b"row length"),
    (dict(hidden=40), b"multiple of 32"), (dict(q=None), b"go together"), (dict(s=None), b"go together"),
    (dict(x=None), b"required"), (dict(h=None, y=None, q=None, s=None), b"required"),
    (dict(x=A + 8), b"aligned"), (dict(residual=B + 2), b"aligned"), (dict(w=D + 4), b"aligned"), (dict(h=E + 8), b"aligned"),
    (dict(y=F + 8), b"aligned"), (dict(q=G + 8), b"aligned"),
    (dict(h=E, y=E), b"two outputs"), (dict(h=E, y=E + 16), b"two outputs"), (dict(q=G, s=G + 255), b"two outputs"),
    (dict(h=A + 16), b"without being it"), (dict(y=B + 496), b"without being it"), (dict(q=A), b"without being it"),
    (dict(s=B + 511), b"without being it"), (dict(y=D), b"weight"),
])
def test_add_rms_norm_refuses(kw, needle):
    refused(norm(**kw), needle)


def product(xq=A, xs=B, m=4, w=D, ws=E, biases=None, n_out=64, n_in=64, y=F, scratch=G, nb=256):
    qt = _lib.QTensor(w, ws, biases, 1.0)
    return _lib.lib().imx_mxfp8_matmul(xq, xs, m, C.byref(qt), n_out, n_in, y, scratch, nb, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(m=-1), b"sizes"), (dict(n_out=0), b"sizes"), (dict(n_in=0), b"sizes"), (dict(n_in=48), b"multiple of 32"),
    (dict(m=0x7fffff80), b"at most"), (dict(n_out=0x7fffffff), b"at most"),
    (dict(n_in=0x7fffffe0), b"at most"), (dict(n_in=0x7fffff20), b"at most"),
    (dict(xq=None), b"required"), (dict(xs=None), b"required"), (dict(w=None), b"required"), (dict(ws=None), b"required"),
    (dict(y=None), b"required"), (dict(biases=A), b"biases"), (dict(xq=A + 4), b"aligned"), (dict(w=D + 8), b"aligned"),
    (dict(y=F + 1), b"aligned"), (dict(y=A + 128), b"overlaps"), (dict(y=B), b"overlaps"), (dict(y=D - 2), b"overlaps"),
    (dict(y=E + 2), b"overlaps"), (dict(y=G), b"overlaps"),
])
def test_mxfp8_matmul_refuses(kw, needle):
    refused(product(**kw), needle)


@pytest.mark.parametrize("kw", [dict(scratch=None), dict(scratch=G + 128), dict(nb=255)])
def test_mxfp8_matmul_refuses_scratch(kw):
    refused(product(**kw), b"scratch", _lib.ERR_WORKSPACE)


def low_rank(y=A, x=B, n=4, n_in=64, a=D, b=D + 0x1000000, scale=None, count=3, rank=8, ids=E, n_out=64, out=F, scratch=G, nb=256):
    ad = _lib.Adapters(a, b, scale, count, rank)
    return _lib.lib().imx_low_rank_add(y, x, n, n_in, C.byref(ad), ids, n_out, out, scratch, nb, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(n=-1), b"sizes"), (dict(n_in=0), b"sizes"), (dict(n_in=60), b"multiple of 8"), (dict(n_out=0), b"sizes"),
    (dict(n_in=(1 << 30) + 8), b"at most"), (dict(n_out=(1 << 30) + 1), b"at most"),
    (dict(y=None), b"required"), (dict(x=None), b"required"), (dict(ids=None), b"required"), (dict(out=None), b"required"),
    (dict(a=None), b"adapter"), (dict(b=None), b"adapter"), (dict(count=0), b"adapter"),
    (dict(rank=0), b"rank"), (dict(rank=12), b"rank"), (dict(rank=264), b"rank"),
    (dict(x=B + 8), b"aligned"), (dict(a=D + 2), b"aligned"), (dict(b=D + 0x1000008), b"aligned"), (dict(y=A + 1), b"aligned"),
    (dict(out=F + 1), b"aligned"), (dict(ids=E + 2), b"aligned"), (dict(out=A + 2), b"without being it"), (dict(out=B), b"overlaps"),
    (dict(out=E), b"overlaps"), (dict(out=D + 16), b"overlaps"), (dict(out=D + 0x1000010), b"overlaps"),
    (dict(scale=F + 4), b"overlaps"), (dict(out=G), b"overlaps"),
])
def test_low_rank_add_refuses(kw, needle):
    refused(low_rank(**kw), needle)


@pytest.mark.parametrize("kw", [dict(scratch=None), dict(scratch=G + 64), dict(nb=0)])
def test_low_rank_add_refuses_scratch(kw):
    refused(low_rank(**kw), b"scratch", _lib.ERR_WORKSPACE)


def test_no_rows_are_no_work():
    """Nothing is read or launched for an empty batch, whose tensors have no address."""
    assert norm(n=0, x=None, residual=None, h=None, y=None, q=None, s=None) == 0
    assert product(m=0, xq=None, xs=None, y=None) == 0
    assert low_rank(n=0, y=None, x=None, ids=None, out=None) == 0


def test_status_block_refuses_no_address():
    refused(_lib.lib().imx_status_block(None), b"nowhere")


def test_scratch_sizes():
    nb = C.c_size_t(0)
    lib = _lib.lib()
    assert lib.imx_mxfp8_matmul_scratch_bytes(5, 100, 64, C.byref(nb)) == 0 and nb.value >= 256
    refused(lib.imx_mxfp8_matmul_scratch_bytes(5, 100, 60, C.byref(nb)), b"bad arguments")
    refused(lib.imx_mxfp8_matmul_scratch_bytes(5, 100, 64, None), b"bad arguments")
    assert lib.imx_low_rank_scratch_bytes(5, 64, 64, 2, 8, C.byref(nb)) == 0 and nb.value >= 256
    refused(lib.imx_low_rank_scratch_bytes(5, 64, 64, 0, 8, C.byref(nb)), b"bad arguments")
    refused(lib.imx_low_rank_scratch_bytes(5, 64, 64, 1, 512, C.byref(nb)), b"bad arguments")


def test_more_rows_than_an_int_counts():
    x = torch.empty(1, 8, device="meta")
    assert ops._row_count("op", x.expand(0x7fffffff, 8), 8) == 0x7fffffff
    with pytest.raises(_lib.IronMLXError, match="rows"):
        ops._row_count("op", x.expand(1 << 31, 8), 8)


def test_dimensions_that_an_int_does_not_hold(monkeypatch):
    """The C ABI takes ints, and ctypes would pass 2^32 + 64 on as 64."""
    monkeypatch.setattr(ops, "_require_same_device", lambda name, *tensors: None)
    monkeypatch.setattr(ops, "_elsewhere", lambda x, stream: False)

    def meta(dtype, *shape):
        return torch.empty(1, device="meta", dtype=dtype).expand(*shape)

    bf, i32, u8 = torch.bfloat16, torch.int32, torch.uint8
    long = 2 ** 32 + 64
    with pytest.raises(_lib.IronMLXError, match="row length"):
        ops.add_rms_norm(meta(bf, 1, long), None, None, 1e-6)
    with pytest.raises(_lib.IronMLXError, match="input dimension"):
        ops.mxfp8_matmul((meta(i32, 1, long // 4), meta(u8, 1, long // 32)), meta(i32, 8, long // 4), meta(u8, 8, long // 32))
    with pytest.raises(_lib.IronMLXError, match="output dimension"):
        ops.mxfp8_matmul((meta(i32, 1, 16), meta(u8, 1, 2)), meta(i32, long, 16), meta(u8, long, 2))
    ids = meta(i32, 1)
    with pytest.raises(_lib.IronMLXError, match="input dimension"):
        ops.low_rank_add(meta(bf, 1, 64), meta(bf, 1, long), meta(bf, 2, 8, long), meta(bf, 2, 64, 8), ids)
    with pytest.raises(_lib.IronMLXError, match="output dimension"):
        ops.low_rank_add(meta(bf, 1, long), meta(bf, 1, 64), meta(bf, 2, 8, 64), meta(bf, 2, long, 8), ids)
    with pytest.raises(_lib.IronMLXError, match="number of adapters"):
        ops.low_rank_add(meta(bf, 1, 64), meta(bf, 1, 64), meta(bf, long, 8, 64), meta(bf, long, 64, 8), ids)
    with pytest.raises(_lib.IronMLXError, match="a rank"):
        ops.low_rank_add(meta(bf, 1, 64), meta(bf, 1, 64), meta(bf, 2, long, 64), meta(bf, 2, 64, long), ids)


def build_cpp(out_dir, name="operators_main"):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe, cuda, lib_dir = os.path.join(out_dir, name), os.environ.get("CUDA_HOME", "/usr/local/cuda"), os.path.dirname(_lib.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(root, "include"), "-I", os.path.join(cuda, "include"),
                    os.path.join(root, "tests", "cpp", name + ".cpp"), "-o", exe, "-L", lib_dir, "-l:libironmlx_b200.so",
                    "-L", os.path.join(cuda, "lib64"), "-lcudart", f"-Wl,-rpath,{lib_dir}", f"-Wl,-rpath,{os.path.join(cuda, 'lib64')}"],
                   check=True, capture_output=True, text=True)
    return exe


def test_cpp_mirror_refuses_shapes(tmp_path):
    if shutil.which("g++") is None or not os.path.exists(_lib.LIB_PATH):
        pytest.skip("g++ or the library is missing")
    done = subprocess.run([build_cpp(str(tmp_path)), "refuse"], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


def test_cpp_mirror_refuses_sizes_that_an_int_does_not_hold(tmp_path):
    if shutil.which("g++") is None or not os.path.exists(_lib.LIB_PATH):
        pytest.skip("g++ or the library is missing")
    done = subprocess.run([build_cpp(str(tmp_path), "operators_sizes_main")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.gpu
def test_cpp_mirror_runs_the_operators(cuda, tmp_path):
    done = subprocess.run([build_cpp(str(tmp_path)), "run"], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.gpu
def test_cpp_mirror_captures_first_calls(cuda, tmp_path):
    done = subprocess.run([build_cpp(str(tmp_path), "operators_capture_main")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


def test_streams_of_another_device():
    class Stream:
        device_index = 1

    class Tensor:
        device = "cuda:0"

        def get_device(self):
            return 0

    with pytest.raises(_lib.IronMLXError, match="stream"):
        ops._on(Tensor(), Stream())


def test_python_layer_refuses_host_tensors_and_other_formats():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    ids = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(_lib.IronMLXError):
        ops.add_rms_norm(x, None, None, 1e-6)
    with pytest.raises(_lib.IronMLXError):
        ops.low_rank_add(x, x, torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 64, 8, dtype=torch.bfloat16), ids)
    w, s = torch.zeros(4, 16, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.uint8)
    with pytest.raises(_lib.IronMLXError):
        ops.mxfp8_matmul((w, s), w, s)
    with pytest.raises(_lib.IronMLXError):
        nn.QuantizedLinear(w, s, None, 64, 4, "affine").forward_rows((w, s))


def test_projection_with_adapters_refuses_host_tensors():
    x, ids = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    adapters = nn.LowRankAdapters(torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 16, 8, dtype=torch.bfloat16))
    for layer in (nn.Linear(torch.zeros(16, 64, dtype=torch.bfloat16)),
                  nn.QuantizedLinear(torch.zeros(16, 16, dtype=torch.int32), torch.zeros(16, 2, dtype=torch.uint8), None, 32, 8, "mxfp8")):
        with pytest.raises(_lib.IronMLXError, match="CUDA"):
            layer.forward_with_adapters(x, adapters, ids)
