"""Answers from posterior draws, on torch tensors of a GPU (include/mhlik.h, "answers from posterior draws").

`quantize` holds rows in 8 bits, `product` gives the predictor x_i.theta_s of every row under every draw, `draw` picks a
column of each row of log weights by a given random number; `PosteriorPredictive` is the three together for the draws a
sampler has kept.  Work is queued on the tensors' GPU, on torch's current stream there; nothing waits for it.  None of
it has gradients: inputs that require them are refused while gradients are recorded, and so are forward-mode tensors with
a tangent.
"""
import ctypes as C
import functools

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib as L

BLOCK = 128

_TYPES = {torch.float64: L.T_F64, torch.float32: L.T_F32, torch.bfloat16: L.T_BF16, torch.float16: L.T_F16}
_OUT = {torch.float32: L.T_F32, torch.bfloat16: L.T_BF16, torch.float16: L.T_F16}
_U = {torch.float64: L.T_F64, torch.float32: L.T_F32}
_E4M3 = {torch.float8_e4m3fn: L.T_Q8}
_CODE = {torch.uint8: None}

_grad = torch.is_grad_enabled


def _chk(rc):
    if rc != 0:
        raise L.MhlikError(rc, (L.load_mhlik().mhlik_last_error(None) or b"").decode())


def _need(ok, text, *args):
    if not ok:
        raise ValueError(text % args if args else text)


def _dual(t):
    return forward_ad.unpack_dual(t).tangent is not None


def _given(name, t, dims, types):
    """The tensor's device, after the checks that every argument has to pass."""
    if (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == dims and t.dtype in types and not (t.requires_grad and _grad())
            and (getattr(forward_ad, "_current_level", 0) < 0 or not _dual(t))):  # outside forward_ad.dual_level there are no tangents
        return t.device
    _need(isinstance(t, torch.Tensor), "%s must be a tensor", name)
    _need(t.is_cuda, "%s must be on a GPU: there is no CPU path", name)
    _need(t.dim() == dims, "%s must have %d dimension(s), not %d", name, dims, t.dim())
    _need(t.dtype in types, "%s has type %s; wanted: %s", name, t.dtype, ", ".join(str(x) for x in types))
    _need(not _dual(t), "%s has a tangent, and there is no gradient: detach it", name)
    raise ValueError("%s requires a gradient, and there is none: detach it" % name)


def _plain(t):
    """t, whose memory holds its values as they are: torch keeps the sign of, for one, c.conj().imag as a mark only."""
    return t.resolve_neg() if t.is_neg() else t


def _same(name, device, wanted):
    if device != wanted:
        raise ValueError("%s is on %s, the rest on %s" % (name, device, wanted))


# The current stream's handle without building a Stream object (a call costs 2 us otherwise); both say the same.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


class Block8:
    """Rows of `cols` values in 8 bits: `data` float8_e4m3fn [rows, 128 ceil(cols / 128)], columns past the last 0, and
    `scale` uint8 [rows, 4 ceil(cols / 512)]: the 128 columns of block b stand for data * 2^(scale[:, b] - 127), with
    scales from 31 to 246 (not checked, which would wait for the GPU; others give wrong products)."""

    __slots__ = ("data", "scale", "cols", "rows", "device")

    def __init__(self, data, scale, cols):
        device = _given("data", data, 2, _E4M3)
        _same("scale", _given("scale", scale, 2, _CODE), device)
        rows, wide = data.shape
        blocks = -(-cols // BLOCK)
        _need(cols >= 1, "cols must be at least 1, not %d", cols)
        _need(wide == blocks * BLOCK, "data has %d columns; %d are %d in blocks of %d", wide, cols, blocks * BLOCK, BLOCK)
        if scale.shape != (rows, (blocks + 3) // 4 * 4):
            raise ValueError("scale has shape %s; wanted %s" % (tuple(scale.shape), (rows, (blocks + 3) // 4 * 4)))
        _need(data.is_contiguous() and scale.is_contiguous(), "data and scale must be contiguous")
        _need(data.data_ptr() % 16 == 0, "data must start at a multiple of 16 bytes")
        _need(scale.data_ptr() % 4 == 0, "scale must start at a multiple of 4 bytes")
        self.data, self.scale, self.cols, self.rows, self.device = data, scale, int(cols), rows, device

    def dequantize(self):
        """The values the rows stand for, as float32 [rows, cols]."""
        blocks = self.data.shape[1] // BLOCK
        step = torch.ldexp(torch.ones((), device=self.device), self.scale[:, :blocks].int() - 127)
        return (self.data.float().view(self.rows, blocks, BLOCK) * step[:, :, None]).view(self.data.shape)[:, : self.cols]


def quantize(x):
    """Rows x [rows, cols] (float64, float32, bfloat16 or float16; any strides) as Block8: each value is rounded once, to
    the nearest e4m3 value on the scale of its block.  What is not finite, or above 448 * 2^119, becomes NaN."""
    device = _given("x", x, 2, _TYPES)
    rows, cols = x.shape
    _need(cols >= 1, "x must have at least one column")
    x = _plain(x)
    blocks = -(-cols // BLOCK)
    q = Block8.__new__(Block8)  # as its constructor would have it
    q.data = torch.empty((rows, blocks * BLOCK), dtype=torch.float8_e4m3fn, device=device)
    q.scale = torch.empty((rows, (blocks + 3) // 4 * 4), dtype=torch.uint8, device=device)
    q.cols, q.rows, q.device = cols, rows, device
    rs, cs = x.stride()
    index = device.index
    _chk(L.load_mhlik().mhlik_q8_quantize(x.data_ptr(), _TYPES[x.dtype], rows, cols, rs, cs, q.data.data_ptr(), q.scale.data_ptr(),
                                          index, _stream(index)))
    return q


@functools.lru_cache(maxsize=256)
def _product_space(rows, cols):
    need = C.c_size_t()
    _chk(L.load_mhlik().mhlik_q8_product_workspace(rows, cols, C.byref(need)))
    return need.value


def product(x, w, dtype=torch.float32):
    """x [rows, cols] (Block8, or values: then quantized here) times the transpose of w (Block8 [draws, cols]): a
    [rows, draws] tensor of `dtype`.  float32 has the accuracy of float32 products and sums; bfloat16 and float16 run at
    the 8-bit matrix rate from 65 rows on, 1.6e-5 of the result's norm off before they are rounded (a hundredth of
    bfloat16's rounding, a tenth of float16's; more of a result that is small against its products)."""
    _need(isinstance(w, Block8), "w must be a Block8 (quantize it once)")
    _need(dtype in _OUT, "dtype is %s; wanted: %s", dtype, ", ".join(str(t) for t in _OUT))
    p = L.Q8Operands()
    device = w.device
    if isinstance(x, Block8):
        _same("x", x.device, device)
        rows, cols = x.rows, x.cols
        p.x, p.x_scale, p.x_type = x.data.data_ptr(), x.scale.data_ptr(), L.T_Q8
    else:
        _same("x", _given("x", x, 2, _TYPES), device)
        rows, cols = x.shape
        x = _plain(x)
        p.x, p.x_type = x.data_ptr(), _TYPES[x.dtype]
        p.x_row_stride, p.x_col_stride = x.stride()
    if cols != w.cols:
        raise ValueError("x has %d columns, w has %d" % (cols, w.cols))
    if p.x_type != L.T_Q8:
        need = _product_space(rows, cols)
        if need:
            space = torch.empty(need, dtype=torch.uint8, device=device)
            p.workspace, p.workspace_bytes = space.data_ptr(), need
    draws = w.rows
    out = torch.empty((rows, draws), dtype=dtype, device=device)
    p.w_data, p.w_scale, p.out = w.data.data_ptr(), w.scale.data_ptr(), out.data_ptr()
    p.out_stride, p.out_type = draws, _OUT[dtype]
    p.rows, p.draws, p.cols = rows, draws, cols
    index = device.index
    _chk(L.load_mhlik().mhlik_q8_product(C.byref(p), index, _stream(index)))
    return out


def _each(name, value, kind, rows, device):
    """A choice that every row has its own of."""
    _same(name, _given(name, value, 1, kind), device)
    _need(value.shape[0] == rows, "%s has %d values for %d rows", name, value.shape[0], rows)
    return _plain(value).contiguous()


_F32, _I32 = {torch.float32: None}, {torch.int32: None}


@functools.lru_cache(maxsize=256)
def _draw_space(rows, n):
    need = C.c_size_t()
    _chk(L.load_mhlik().mhlik_draw_workspace(rows, n, C.byref(need)))
    return need.value


def draw(z, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """One column of each row of log weights z [rows, n] (float32, bfloat16, float16), by the random numbers u [rows] in
    [0, 1) (float64 or float32): (column int64 [rows], its log probability float32 [rows]).

    Weights are exp((z - max) / temperature), +inf counting as the largest float; of them the top_k largest are kept, of
    these the fewest that hold top_p of their mass, of these the ones at least min_p times the largest; equal weights keep
    the lower columns. The column is the first, in column order, at which the kept mass exceeds u of the whole.
    temperature 0 takes the largest. The four choices are numbers, or tensors of one value a row (float32; top_k int32);
    None is off, and so are top_k <= 0, top_p >= 1, min_p <= 0. A row with nothing to draw (all -inf, or a NaN) gives
    column -1 and NaN."""
    device = _given("z", z, 2, _OUT)
    _same("u", _given("u", u, 1, _U), device)
    rows, n = z.shape
    _need(n >= 1, "z must have at least one column")
    _need(u.shape[0] == rows, "u has %d values for %d rows", u.shape[0], rows)
    z, u = _plain(z), _plain(u)
    stride, step = z.stride()
    if step != 1 and n > 1:
        z = z.contiguous()
        stride = n
    if not u.is_contiguous():
        u = u.contiguous()
    p = L.DrawRows()
    if isinstance(temperature, torch.Tensor):
        temperature = _each("temperature", temperature, _F32, rows, device)
        p.temperature = temperature.data_ptr()
    else:
        p.temperature_all = 1.0 if temperature is None else temperature
    if isinstance(top_k, torch.Tensor):
        top_k = _each("top_k", top_k, _I32, rows, device)
        p.top_k = top_k.data_ptr()
    elif top_k is not None:
        p.top_k_all = max(0, min(top_k, n))
    if isinstance(top_p, torch.Tensor):
        top_p = _each("top_p", top_p, _F32, rows, device)
        p.top_p = top_p.data_ptr()
    else:
        p.top_p_all = 1.0 if top_p is None else top_p
    if isinstance(min_p, torch.Tensor):
        min_p = _each("min_p", min_p, _F32, rows, device)
        p.min_p = min_p.data_ptr()
    elif min_p is not None:
        p.min_p_all = min_p
    index = torch.empty(rows, dtype=torch.int64, device=device)
    logp = torch.empty(rows, dtype=torch.float32, device=device)
    p.z, p.rows, p.n, p.stride, p.z_type = z.data_ptr(), rows, n, stride, _OUT[z.dtype]
    p.u, p.u_type = u.data_ptr(), _U[u.dtype]
    p.index, p.logp = index.data_ptr(), logp.data_ptr()
    need = _draw_space(rows, n)
    if need:
        space = torch.empty(need, dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = space.data_ptr(), need
    gpu = device.index
    _chk(L.load_mhlik().mhlik_draw(C.byref(p), gpu, _stream(gpu)))
    return index, logp


class PosteriorPredictive:
    """New observations under the draws that a sampler has kept: theta [draws, cols] (the `samples` of a sampler, or a
    tensor), held in 8 bits on one GPU.

    A predictor x.theta_s differs from the one in 32 bits by the rounding of x and theta_s to four significant bits, 2^-4
    relative for each product at most and of either sign, so that averages over draws and columns lose most of it.  An
    accept test would not: the samplers' likelihoods do not go through here."""

    CHUNK = 1 << 26  # predictors held at a time

    def __init__(self, theta, device=None):
        theta = torch.as_tensor(theta)
        if not theta.is_cuda or device is not None:
            theta = theta.to("cuda" if device is None else device)
        _need(theta.dim() == 2 and theta.shape[0] >= 1, "theta must have two dimensions and at least one draw")
        self.theta = quantize(theta.detach())

    def predictor(self, x, dtype=torch.float32):
        """x_i.theta_s for every row of x [rows, cols] and every draw."""
        return product(x, self.theta, dtype)

    def _chunks(self, rows):
        step = max(1, self.CHUNK // self.theta.rows)
        return ((i, min(rows, i + step)) for i in range(0, rows, step))

    def probability(self, x):
        """P(y = 1 | x_i), float32 [rows]: the mean of 1 / (1 + exp(-x_i.theta_s)) over the draws."""
        _given("x", x, 2, _TYPES)
        out = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
        for i, j in self._chunks(x.shape[0]):
            torch.mean(torch.sigmoid(self.predictor(x[i:j])), 1, out=out[i:j])
        return out

    def case_deletion(self, x, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
        """For every observation a draw from the posterior without it: (draw int64 [rows], log probability [rows]).

        x holds the observations with their labels folded in, as the samplers' design matrix does (-y_i x_i): then
        1 / p(y_i | x_i, theta_s) = 1 + exp(x_i.theta_s) are the weights that take observation i out of the posterior.
        u [rows] are random numbers in [0, 1); the other arguments flatten or cut the weights, see `draw`."""
        _given("x", x, 2, _TYPES)
        rows = x.shape[0]
        _same("u", _given("u", u, 1, _U), x.device)
        _need(u.shape[0] == rows, "u has %d values for %d rows", u.shape[0], rows)
        choices = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
        for name, value in choices.items():
            if isinstance(value, torch.Tensor):
                _each(name, value, _I32 if name == "top_k" else _F32, rows, x.device)
        index = torch.empty(rows, dtype=torch.int64, device=x.device)
        logp = torch.empty(rows, dtype=torch.float32, device=x.device)
        zero = torch.zeros((), device=x.device)
        for i, j in self._chunks(rows):
            part = {k: v[i:j] if isinstance(v, torch.Tensor) else v for k, v in choices.items()}
            index[i:j], logp[i:j] = draw(torch.logaddexp(self.predictor(x[i:j]), zero), u[i:j], **part)
        return index, logp
