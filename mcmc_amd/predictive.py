"""Answers from posterior draws, on torch tensors of a GPU (include/mhlik.h, "answers from posterior draws").

`quantize` holds rows in 8 bits, `product` gives the predictor x_i.theta_s of every row under every draw, `draw` picks a
column of each row of log weights by a given random number; `PosteriorPredictive` is the three together for the draws a
sampler has kept.  Work is queued on the tensors' GPU, on torch's current stream there; nothing waits for it.  None of
it has gradients: inputs that require them are refused while gradients are recorded.
"""
import ctypes as C

import torch

from . import _lib as L

BLOCK = 128

_TYPES = {torch.float64: L.T_F64, torch.float32: L.T_F32, torch.bfloat16: L.T_BF16, torch.float16: L.T_F16}
_OUT = {torch.float32: L.T_F32, torch.bfloat16: L.T_BF16, torch.float16: L.T_F16}
_U = {torch.float64: L.T_F64, torch.float32: L.T_F32}


def _chk(rc):
    if rc != 0:
        raise L.MhlikError(rc, (L.load_mhlik().mhlik_last_error(None) or b"").decode())


def _need(ok, text, *args):
    if not ok:
        raise ValueError(text % args if args else text)


def _given(name, t, dims, types):
    _need(isinstance(t, torch.Tensor), "%s must be a tensor", name)
    _need(t.is_cuda, "%s must be on a GPU: there is no CPU path", name)
    _need(t.dim() == dims, "%s must have %d dimension(s), not %d", name, dims, t.dim())
    _need(t.dtype in types, "%s has type %s; wanted: %s", name, t.dtype, ", ".join(str(x) for x in types))
    _need(not (t.requires_grad and torch.is_grad_enabled()), "%s requires a gradient, and there is none: detach it", name)


def _same(name, t, device):
    _need(t.device == device, "%s is on %s, the rest on %s", name, t.device, device)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


class Block8:
    """Rows of `cols` values in 8 bits: `data` float8_e4m3fn [rows, 128 ceil(cols / 128)], columns past the last 0, and
    `scale` uint8 [rows, 4 ceil(cols / 512)]: the 128 columns of block b stand for data * 2^(scale[:, b] - 127)."""

    __slots__ = ("data", "scale", "cols")

    def __init__(self, data, scale, cols):
        _given("data", data, 2, (torch.float8_e4m3fn,))
        _given("scale", scale, 2, (torch.uint8,))
        _same("scale", scale, data.device)
        blocks = -(-cols // BLOCK)
        _need(cols >= 1, "cols must be at least 1, not %d", cols)
        _need(data.shape[1] == blocks * BLOCK, "data has %d columns; %d are %d in blocks of %d", data.shape[1], cols, blocks * BLOCK, BLOCK)
        _need(tuple(scale.shape) == (data.shape[0], 4 * -(-blocks // 4)), "scale has shape %s; wanted %s", tuple(scale.shape),
              (data.shape[0], 4 * -(-blocks // 4)))
        _need(data.is_contiguous() and scale.is_contiguous(), "data and scale must be contiguous")
        _need(data.data_ptr() % 16 == 0, "data must start at a multiple of 16 bytes")
        self.data, self.scale, self.cols = data, scale, int(cols)

    @property
    def rows(self):
        return self.data.shape[0]

    def dequantize(self):
        """The values the rows stand for, as float32 [rows, cols]."""
        blocks = self.data.shape[1] // BLOCK
        step = torch.ldexp(torch.ones((), device=self.data.device), self.scale[:, :blocks].int() - 127)
        return (self.data.float().view(-1, blocks, BLOCK) * step[:, :, None]).view(self.data.shape)[:, : self.cols]


def _empty8(rows, cols, device):
    blocks = -(-cols // BLOCK)
    return (torch.empty(rows, blocks * BLOCK, dtype=torch.float8_e4m3fn, device=device),
            torch.empty(rows, 4 * -(-blocks // 4), dtype=torch.uint8, device=device))


def quantize(x):
    """Rows x [rows, cols] (float64, float32, bfloat16 or float16; any strides) as Block8: each value is rounded once, to
    the nearest e4m3 value on the scale of its block.  What is not finite, or above 448 * 2^119, becomes NaN."""
    _given("x", x, 2, _TYPES)
    rows, cols = x.shape
    _need(cols >= 1, "x must have at least one column")
    data, scale = _empty8(rows, cols, x.device)
    rs, cs = x.stride()
    _chk(L.load_mhlik().mhlik_q8_quantize(x.data_ptr(), _TYPES[x.dtype], rows, cols, rs, cs, data.data_ptr(), scale.data_ptr(),
                                          x.device.index, _stream(x.device)))
    return Block8(data, scale, cols)


def product(x, w, dtype=torch.float32):
    """x [rows, cols] (Block8, or values: then quantized here) times the transpose of w (Block8 [draws, cols]): a
    [rows, draws] tensor of `dtype`.  float32 has the accuracy of float32 products and sums; bfloat16 and float16 run at
    the 8-bit matrix rate, 1.6e-5 of the result's norm off before they are rounded."""
    _need(isinstance(w, Block8), "w must be a Block8 (quantize it once)")
    _need(dtype in _OUT, "dtype is %s; wanted: %s", dtype, ", ".join(str(t) for t in _OUT))
    p = L.Q8Operands()
    device = w.data.device
    if isinstance(x, Block8):
        _same("x", x.data, device)
        rows, cols = x.rows, x.cols
        p.x, p.x_scale, p.x_type = x.data.data_ptr(), x.scale.data_ptr(), L.T_Q8
    else:
        _given("x", x, 2, _TYPES)
        _same("x", x, device)
        rows, cols = x.shape
        p.x, p.x_type = x.data_ptr(), _TYPES[x.dtype]
        p.x_row_stride, p.x_col_stride = x.stride()
    _need(cols == w.cols, "x has %d columns, w has %d", cols, w.cols)
    if p.x_type != L.T_Q8:
        p.workspace_bytes = rows * (w.data.shape[1] + w.scale.shape[1])
        space = torch.empty(p.workspace_bytes, dtype=torch.uint8, device=device)
        p.workspace = space.data_ptr()
    out = torch.empty(rows, w.rows, dtype=dtype, device=device)
    p.w_data, p.w_scale, p.out = w.data.data_ptr(), w.scale.data_ptr(), out.data_ptr()
    p.out_stride, p.out_type = w.rows, _OUT[dtype]
    p.rows, p.draws, p.cols = rows, w.rows, cols
    _chk(L.load_mhlik().mhlik_q8_product(C.byref(p), device.index, _stream(device)))
    return out


def _choice(p, name, value, off, dtype, rows, device, held):
    if value is None:
        value = off
    if isinstance(value, torch.Tensor):
        _given(name, value, 1, (dtype,))
        _same(name, value, device)
        _need(value.shape[0] == rows, "%s has %d values for %d rows", name, value.shape[0], rows)
        value = value.contiguous()
        held.append(value)
        setattr(p, name, value.data_ptr())
    else:
        setattr(p, name + "_all", value)


def draw(z, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """One column of each row of log weights z [rows, n] (float32, bfloat16, float16), by the random numbers u [rows] in
    [0, 1) (float64 or float32): (column int64 [rows], its log probability float32 [rows]).

    Weights are exp((z - max) / temperature); of them the top_k largest are kept, of these the fewest that hold top_p of
    their mass, of these the ones at least min_p times the largest; equal weights keep the lower columns.  The column is
    the first, in column order, at which the kept mass exceeds u of the whole.  temperature 0 takes the largest.  The
    four choices are numbers, or tensors of one value a row (float32; top_k int32); None is off, and so are top_k <= 0,
    top_p >= 1, min_p <= 0.  A row with nothing to draw (all -inf, or a NaN) gives column -1 and NaN."""
    _given("z", z, 2, _OUT)
    _given("u", u, 1, _U)
    rows, n = z.shape
    device = z.device
    _same("u", u, device)
    _need(n >= 1, "z must have at least one column")
    _need(u.shape[0] == rows, "u has %d values for %d rows", u.shape[0], rows)
    if z.stride(1) != 1 and n > 1:
        z = z.contiguous()
    u = u.contiguous()
    p = L.DrawRows()
    held = []
    _choice(p, "temperature", temperature, 1.0, torch.float32, rows, device, held)
    _choice(p, "top_k", top_k, 0, torch.int32, rows, device, held)
    _choice(p, "top_p", top_p, 1.0, torch.float32, rows, device, held)
    _choice(p, "min_p", min_p, 0.0, torch.float32, rows, device, held)
    index = torch.empty(rows, dtype=torch.int64, device=device)
    logp = torch.empty(rows, dtype=torch.float32, device=device)
    p.z, p.rows, p.n, p.stride, p.z_type = z.data_ptr(), rows, n, z.stride(0), _OUT[z.dtype]
    p.u, p.u_type = u.data_ptr(), _U[u.dtype]
    p.index, p.logp = index.data_ptr(), logp.data_ptr()
    need = C.c_size_t()
    _chk(L.load_mhlik().mhlik_draw_workspace(rows, n, C.byref(need)))
    if need.value:
        space = torch.empty(need.value, dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = space.data_ptr(), need.value
    _chk(L.load_mhlik().mhlik_draw(C.byref(p), device.index, _stream(device)))
    return index, logp
