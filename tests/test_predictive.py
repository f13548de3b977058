"""The predictive operators' interface without a GPU: what the C calls and the Python layer refuse before any device is
touched, the sizes they state, and the structs' layouts."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20  # an aligned address that no refused call may touch


@pytest.fixture(scope="module")
def lib():
    from mcmc_amd import _lib

    return _lib.load_mhlik()


def _refused(lib, rc, text):
    assert rc == 1, rc  # MHLIK_EINVAL
    assert text in lib.mhlik_last_error(None).decode()


@pytest.mark.parametrize("change,text", [
    (dict(type=0), "unknown element type"), (dict(type=9), "unknown element type"), (dict(rows=-1), "0 <= rows"),
    (dict(cols=0), "1 <= cols"), (dict(cols=(1 << 22) + 1), "1 <= cols"), (dict(rows=(1 << 40) + 1), "0 <= rows"),
    (dict(x=None), "x must not be NULL"), (dict(x=FAKE + 2), "not aligned to its type"), (dict(rs=-1), "strides must not be negative"),
    (dict(cs=-4), "strides must not be negative"), (dict(data=None), "must not be NULL"), (dict(scale=None), "must not be NULL"),
    (dict(data=FAKE + 8), "multiple of 16 bytes"), (dict(scale=FAKE + 2), "multiple of 4 bytes"),
])
def test_quantize_refuses(lib, change, text):
    a = dict(x=FAKE, type=2, rows=4, cols=100, rs=100, cs=1, data=FAKE, scale=FAKE)
    a.update(change)
    rc = lib.mhlik_q8_quantize(a["x"], a["type"], a["rows"], a["cols"], a["rs"], a["cs"], a["data"], a["scale"], 0, None)
    _refused(lib, rc, text)


def _operands(**change):
    from mcmc_amd import _lib

    a = dict(x=FAKE, x_scale=FAKE, w_data=FAKE, w_scale=FAKE, out=FAKE, out_stride=7, rows=100, draws=7, cols=300, x_type=0, out_type=2)
    a.update(change)
    p = _lib.Q8Operands()
    for k, v in a.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,text", [
    (dict(x_type=7), "unknown element type"), (dict(out_type=0), "out: unknown element type"), (dict(out_type=1), "out: unknown element type"),
    (dict(out_stride=6), "less than draws"), (dict(out=None), "out is NULL"), (dict(out=FAKE + 1), "not aligned"),
    (dict(x=FAKE + 8), "x: data must start"), (dict(w_data=FAKE + 4), "w: data must start"), (dict(w_scale=None), "must not be NULL"),
    (dict(x_scale=None), "must not be NULL"), (dict(cols=0), "1 <= cols"), (dict(draws=-1), "0 <= rows"),
    (dict(x_type=2, x_row_stride=-1), "strides must not be negative"),
    (dict(x_type=2, x=FAKE + 1), "not aligned to its type"),
    (dict(x_type=2), "workspace"), (dict(x_type=2, workspace=FAKE, workspace_bytes=100 * (384 + 4) - 1), "workspace"),
    (dict(x_type=2, workspace=FAKE + 8, workspace_bytes=1 << 20), "workspace"),
    (dict(x_scale=FAKE + 1), "x: scale must start"), (dict(w_scale=FAKE + 2), "w: scale must start"),
])
def test_product_refuses(lib, change, text):
    rc = lib.mhlik_q8_product(C.byref(_operands(**change)), -1, None)
    _refused(lib, rc, text)


def test_product_refuses_no_operands(lib):
    _refused(lib, lib.mhlik_q8_product(None, 0, None), "operands")


def _rows(**change):
    from mcmc_amd import _lib

    a = dict(z=FAKE, rows=3, n=10, stride=10, u=FAKE, temperature_all=1.0, top_p_all=1.0, min_p_all=0.0, index=FAKE, logp=FAKE,
             top_k_all=0, z_type=2, u_type=1)
    a.update(change)
    p = _lib.DrawRows()
    for k, v in a.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,text", [
    (dict(z_type=1), "z: unknown element type"), (dict(z_type=0), "z: unknown element type"), (dict(u_type=3), "u: unknown element type"),
    (dict(n=0), "1 <= n"), (dict(n=1 << 30), "1 <= n"), (dict(rows=-1), "0 <= rows"), (dict(rows=1 << 31), "0 <= rows"),
    (dict(z=None), "z must not be NULL"), (dict(z=FAKE + 2), "not aligned"), (dict(stride=-1), "strides"), (dict(u=None), "u and index"),
    (dict(index=None), "u and index"), (dict(temperature_all=-1.0), "temperature"), (dict(temperature_all=1e-200), "temperature"),
    (dict(temperature_all=float("nan")), "temperature"), (dict(top_p_all=float("nan")), "top_p"), (dict(min_p_all=float("nan")), "min_p"),
    (dict(n=9000, stride=9000), "workspace"), (dict(n=9000, stride=9000, workspace=FAKE, workspace_bytes=100), "workspace"),
])
def test_draw_refuses(lib, change, text):
    _refused(lib, lib.mhlik_draw(C.byref(_rows(**change)), 0, None), text)


def test_nothing_to_do_is_no_error(lib):
    """No rows: no pointer is looked at and no device is needed."""
    assert lib.mhlik_q8_quantize(None, 2, 0, 5, 5, 1, None, None, 0, None) == 0
    assert lib.mhlik_q8_product(C.byref(_operands(rows=0, x=None, x_scale=None, out=None)), 0, None) == 0
    assert lib.mhlik_q8_product(C.byref(_operands(draws=0, w_data=None, w_scale=None, out=None)), 0, None) == 0
    assert lib.mhlik_draw(C.byref(_rows(rows=0, z=None, u=None, index=None)), 0, None) == 0


def test_workspace_sizes(lib):
    need = C.c_size_t()
    assert lib.mhlik_q8_product_workspace(100, 300, C.byref(need)) == 0 and need.value == 100 * (384 + 4)
    assert lib.mhlik_q8_product_workspace(64, 256, C.byref(need)) == 0 and need.value == 0  # the product's own kernel takes them
    assert lib.mhlik_q8_product_workspace(65, 10, C.byref(need)) == 0 and need.value == 65 * (128 + 4)
    assert lib.mhlik_q8_product_workspace(1 << 40, 1 << 22, C.byref(need)) == 0 and need.value == (1 << 40) * ((1 << 22) + (1 << 15))
    assert lib.mhlik_draw_workspace(5, 8192, C.byref(need)) == 0 and need.value == 0  # a workgroup holds the row
    assert lib.mhlik_draw_workspace(5, 8193, C.byref(need)) == 0 and need.value > 0
    a = need.value
    assert lib.mhlik_draw_workspace(10, 8193, C.byref(need)) == 0 and a < need.value < 2 * a + 4096
    _refused(lib, lib.mhlik_q8_product_workspace(1, 0, C.byref(need)), "cols")
    _refused(lib, lib.mhlik_draw_workspace(1, 10, None), "bytes")
    _refused(lib, lib.mhlik_draw_workspace(1, 0, C.byref(need)), "1 <= n")


def test_the_draw_workspace_is_bounded(lib):
    """Long rows go in parts: however many there are, their workspace stays below 0.75 GB.  It is largest for the shortest
    ones, whose units are the least filled."""
    need = C.c_size_t()
    sizes = {}
    for n in (8193, 8320, 10241, 20001, 65537, 131072, 1 << 20, 1 << 21):
        for rows in (1, 100, 20000, (1 << 31) - 1):
            assert lib.mhlik_draw_workspace(rows, n, C.byref(need)) == 0
            sizes[n, rows] = need.value
    assert max(sizes.values()) == sizes[8193, (1 << 31) - 1] < 750_000_000
    assert lib.mhlik_draw_workspace((1 << 31) - 1, (1 << 21) + 1, C.byref(need)) == 0 and need.value == 0  # no units


def test_struct_layouts_match_the_header():
    from mcmc_amd import _lib

    fields = {"mhlik_q8_operands": _lib.Q8Operands, "mhlik_draw_rows": _lib.DrawRows}
    lines = []
    for name, mirror in fields.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f) for f, _ in mirror._fields_]
    src = '#include "mhlik.h"\n#include <stdio.h>\nint main(void){ %s return 0; }\n' % " ".join(lines)
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "p.c"), os.path.join(td, "p")
        open(c, "w").write(src)
        subprocess.check_call(["gcc", "-I" + os.path.join(ROOT, "include"), c, "-o", exe])
        out = [int(x) for x in subprocess.check_output([exe], text=True).split()]
    want = []
    for mirror in fields.values():
        want += [C.sizeof(mirror)] + [getattr(mirror, f).offset for f, _ in mirror._fields_]
    assert out == want


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="only meaningful without a GPU")
def test_fails_loudly_without_gpu(lib):
    assert lib.mhlik_draw(C.byref(_rows()), 0, None) == 3  # MHLIK_EHIP
    assert "hipGetDevice" in lib.mhlik_last_error(None).decode() or "failed" in lib.mhlik_last_error(None).decode()


def test_python_refuses_cpu_tensors():
    import torch

    from mcmc_amd import predictive as P

    x, z, u = torch.zeros(3, 5), torch.zeros(3, 5), torch.zeros(3)
    for call in (lambda: P.quantize(x), lambda: P.draw(z, u), lambda: P.Block8(torch.zeros(3, 128).to(torch.float8_e4m3fn), torch.zeros(3, 4, dtype=torch.uint8), 5)):
        with pytest.raises(ValueError, match="must be on a GPU"):
            call()
    with pytest.raises(ValueError, match="must be a tensor"):
        P.quantize([[1.0]])
    with pytest.raises(ValueError, match="must be a Block8"):
        P.product(x, x)
