"""fhessm.client -- the client's token step on the GPU.

After a tick the client decrypts one normed row per conversation, applies the tied head in plaintext (--dec-out,
gpu_real_model.cu:2444-2533), picks a token (spec_decode/decode_policy.py:37) and encrypts that
token's row of the same table (ml-eval/fhe_client.py:123-135).  Here the table is held in 4 bits with
a scale for each group of columns, and the three steps are kernels:

  * ``q4_matvec``: logits (or any product with a 4-bit table);
  * ``sample``: temperature, top-k, top-p and min-p from given random numbers;
  * ``q4_rows``: rows of the table by token id;
  * ``TokenHead``: the three together.

Tensors are torch tensors on the context's GPU; calls are enqueued on torch's current stream of that
GPU, like any torch operation, and do not synchronise.  A call that cannot be served raises
``FheError``; nothing is converted or copied silently.
"""
import ctypes as C

import numpy as np
import torch

from . import FheError, _check, lib

_VP = C.c_void_p
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_LEGACY_STREAM = 1      # cudaStreamLegacy: torch calls its default stream 0, which the C-ABI takes for the context's
MAX_VOCAB = 1 << 20


class Q4C(C.Structure):
    _fields_ = [("q", _VP), ("scale", _VP), ("scale_type", C.c_int), ("rows", C.c_int), ("cols", C.c_int),
                ("group", C.c_int), ("ldq", C.c_longlong), ("lds", C.c_longlong)]


class SampleC(C.Structure):
    _fields_ = [("temperature", _VP), ("top_k", _VP), ("top_p", _VP), ("min_p", _VP), ("temperature_all", C.c_float),
                ("top_k_all", C.c_int32), ("top_p_all", C.c_float), ("min_p_all", C.c_float)]


_fns = None


def _sigs():
    global _fns
    if _fns is None:
        h = lib()
        for name, args in [
            ("fhe_q4_matvec", [_VP, C.POINTER(Q4C), _VP, C.c_int, C.c_longlong, C.c_int, _VP, C.c_int, C.c_longlong,
                               _VP]),
            ("fhe_q4_rows", [_VP, C.POINTER(Q4C), _VP, C.c_int, _VP, C.c_int, C.c_longlong, _VP]),
            ("fhe_sample", [_VP, C.POINTER(SampleC), _VP, C.c_int, C.c_longlong, C.c_int, C.c_int, _VP, _VP, _VP, _VP]),
        ]:
            f = getattr(h, name)
            f.restype = C.c_int
            f.argtypes = args
        _fns = h
    return _fns


def _bad(msg):
    return FheError(-1, msg)


def _stream(device):
    # torch.cuda.current_stream(device).cuda_stream without the Stream object, 2 us of a call's 8
    return torch._C._cuda_getCurrentRawStream(device) or _LEGACY_STREAM


def _on_gpu(device, t, what):
    if t.get_device() != device or t.device.type != "cuda":
        raise _bad(f"{what} is not on the context's GPU (cuda:{device})")


def _rows_of(t, what):
    """(type, row count, row length, row stride) of a 2-d tensor with contiguous rows."""
    if t.dim() != 2:
        raise _bad(f"{what}: expected rows x columns, got {tuple(t.shape)}")
    if t.dtype not in _TYPES:
        raise _bad(f"{what}: float32, float16 or bfloat16, got {t.dtype}")
    m, n = t.shape
    if n > 1 and t.stride(1) != 1:
        raise _bad(f"{what}: the values of a row are not contiguous")
    ld = t.stride(0) if m > 1 else n
    if m > 1 and ld < n:
        raise _bad(f"{what}: rows overlap")
    return _TYPES[t.dtype], m, n, ld


class Q4Table:
    """A table of rows x cols values in 4 bits with a scale for each `group` columns of a row:
    value (i, c) = scale[i, c // group] * (q - 8), q the low (even c) or high (odd c) half of byte
    weight[i, c // 2].  weight: uint8 (rows, bytes), a row padded to a multiple of 16 bytes;
    scale: float32, float16 or bfloat16 (rows, ceil(cols / group)); group: a multiple of 32."""

    __slots__ = ("weight", "scale", "rows", "cols", "group", "c", "ref")

    def __init__(self, weight, scale, *, cols, group):
        if weight.dtype != torch.uint8 or weight.dim() != 2:
            raise _bad("q4 table: weight is a uint8 tensor, rows x bytes")
        rows, nbytes = weight.shape
        if cols < 1 or group < 32 or group % 32:
            raise _bad("q4 table: cols >= 1 and group a multiple of 32")
        if nbytes < -(-cols // 32) * 16:
            raise _bad("q4 table: rows are padded to a multiple of 16 bytes (32 columns)")
        st, srows, groups, lds = _rows_of(scale, "q4 scales")
        if srows != rows or groups != -(-cols // group):
            raise _bad(f"q4 scales: expected {(rows, -(-cols // group))}, got {tuple(scale.shape)}")
        if weight.stride(1) != 1:
            raise _bad("q4 table: the bytes of a row are not contiguous")
        if scale.device != weight.device:
            raise _bad("q4 table: weight and scale are on different devices")
        ldq = weight.stride(0) if rows > 1 else -(-nbytes // 16) * 16
        if rows > 1 and ldq < nbytes:
            raise _bad("q4 table: rows overlap")
        self.weight, self.scale, self.rows, self.cols, self.group = weight, scale, rows, cols, group
        self.c = Q4C(weight.data_ptr(), scale.data_ptr(), st, rows, cols, group, ldq, lds)
        self.ref = C.byref(self.c)

    @classmethod
    def quantise(cls, w, *, group=64, scale_dtype=torch.float16, device="cpu"):
        """The 4-bit table nearest to w (rows x cols, a float array or tensor): a group's scale is its largest
        magnitude over 7, rounded to scale_dtype."""
        w = torch.as_tensor(np.asarray(w) if not torch.is_tensor(w) else w).to(device=device, dtype=torch.float32)
        if w.dim() != 2 or group < 32 or group % 32:
            raise _bad("quantise: rows x cols and a group that is a multiple of 32")
        rows, cols = w.shape
        groups = -(-cols // group)
        wide = torch.zeros(rows, groups * group, dtype=torch.float32, device=w.device)
        wide[:, :cols] = w
        wide = wide.view(rows, groups, group)
        scale = (wide.abs().amax(2) / 7).to(scale_dtype)
        s = scale.float().unsqueeze(2)
        q = torch.where(s > 0, torch.round(wide / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(wide))
        q = (q.clamp(-8, 7) + 8).to(torch.uint8).view(rows, -1)[:, :-(-cols // 32) * 32]
        return cls((q[:, 0::2] | q[:, 1::2] << 4).contiguous(), scale.contiguous(), cols=cols, group=group)

    def to(self, device):
        return Q4Table(self.weight.to(device), self.scale.to(device), cols=self.cols, group=self.group)

    def dequantise(self):
        """The table's values, float32 (rows, cols)."""
        q = torch.stack([self.weight & 15, self.weight >> 4], dim=-1).flatten(-2)[:, :self.cols].float() - 8
        return q * self.scale.float().repeat_interleave(self.group, dim=1)[:, :self.cols]


def _out(out, like, shape, dtype, device):
    """(output, its type, its row stride): a new one, or the caller's."""
    if dtype not in _TYPES:
        raise _bad(f"out: float32, float16 or bfloat16, got {dtype}")
    if out is None:
        return like.new_empty(shape, dtype=dtype), _TYPES[dtype], shape[1]
    if tuple(out.shape) != shape or out.dtype != dtype:
        raise _bad(f"out: expected {dtype} {shape}, got {out.dtype} {tuple(out.shape)}")
    _on_gpu(device, out, "out")
    ot, _, _, ldo = _rows_of(out, "out")
    return out, ot, ldo


def q4_matvec(cx, x, table, *, dtype=torch.float32, out=None):
    """x (m, cols) times the table's transpose: (m, rows) of `dtype` (fhe_q4_matvec).  x: float32,
    float16 or bfloat16 with contiguous rows (any row stride)."""
    xt, m, k, ldx = _rows_of(x, "x")
    if k != table.cols:
        raise _bad(f"x has {k} columns, the table {table.cols}")
    device = cx.p.device
    _on_gpu(device, x, "x")
    _on_gpu(device, table.weight, "q4 table")
    out, ot, ldo = _out(out, x, (m, table.rows), dtype, device)
    _check((_fns or _sigs()).fhe_q4_matvec(cx.h, table.ref, x.data_ptr(), xt, ldx, m, out.data_ptr(), ot, ldo,
                                           _stream(device)))
    return out


def q4_rows(cx, tokens, table, *, dtype=torch.float32, out=None):
    """Rows of the table by token id: tokens (m,) int64 -> (m, cols) of `dtype` (fhe_q4_rows); a token
    outside the table (the -1 of an empty row) gives zeros."""
    if tokens.dim() != 1 or tokens.dtype != torch.int64 or (tokens.numel() > 1 and tokens.stride(0) != 1):
        raise _bad("tokens: a contiguous int64 vector")
    device = cx.p.device
    _on_gpu(device, tokens, "tokens")
    _on_gpu(device, table.weight, "q4 table")
    m = tokens.shape[0]
    out, ot, ldo = _out(out, tokens, (m, table.cols), dtype, device)
    _check((_fns or _sigs()).fhe_q4_rows(cx.h, table.ref, tokens.data_ptr(), m, out.data_ptr(), ot, ldo,
                                         _stream(device)))
    return out


def _setting(device, v, rows, dtype, what):
    """(device pointer or None, plain value) of a setting given as one number or as a value per row."""
    if not torch.is_tensor(v):
        return None, v
    if v.dim() != 1 or v.shape[0] != rows or v.dtype != dtype or (rows > 1 and v.stride(0) != 1):
        raise _bad(f"{what}: one number, or a contiguous {dtype} vector with a value for each row")
    _on_gpu(device, v, what)
    return v.data_ptr(), 0


def sample(cx, logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token per row of logits (rows, vocab) from the random numbers u (rows,) in [0, 1): (tokens
    int64, log-probabilities float32) (fhe_sample, whose comment defines the choice).  Each setting is
    one number or a vector with a value for each row (float32; top_k int32).  temperature 0: the
    largest logit.  top_k 0, top_p 1 and min_p 0 are off.  The token of a row that allows none is -1."""
    lt, rows, vocab, ld = _rows_of(logits, "logits")
    device = cx.p.device
    _on_gpu(device, logits, "logits")
    if not 1 <= vocab <= MAX_VOCAB:
        raise _bad(f"logits: a vocabulary of 1 to {MAX_VOCAB}")
    up, _ = _setting(device, u, rows, torch.float32, "u")
    if up is None:
        raise _bad("u: a float32 vector with a random number for each row")
    t, t1 = _setting(device, temperature, rows, torch.float32, "temperature")
    k, k1 = _setting(device, top_k, rows, torch.int32, "top_k")
    p, p1 = _setting(device, top_p, rows, torch.float32, "top_p")
    mp, mp1 = _setting(device, min_p, rows, torch.float32, "min_p")
    token, logprob = u.new_empty(rows, dtype=torch.int64), u.new_empty(rows)
    cfg = SampleC(t, k, p, mp, t1, min(k1, vocab), p1, mp1)
    _check((_fns or _sigs()).fhe_sample(cx.h, C.byref(cfg), logits.data_ptr(), lt, ld, rows, vocab, up,
                                        token.data_ptr(), logprob.data_ptr(), _stream(device)))
    return token, logprob


class TokenHead:
    """The client's side of a decode tick with a tied 4-bit table: decrypted normed rows in, tokens and the
    next tick's input rows out."""

    def __init__(self, cx, table):
        self.cx = cx
        self.table = table.to(f"cuda:{cx.p.device}")

    def logits(self, hidden):
        """hidden (lanes, d): a float32, float16 or bfloat16 tensor on the GPU, or a host array (what
        unpack_lanes gives), which is copied as float32."""
        if not torch.is_tensor(hidden):
            hidden = torch.from_numpy(np.ascontiguousarray(hidden, dtype=np.float32)).to(self.table.weight.device)
        return q4_matvec(self.cx, hidden, self.table)

    def embed(self, tokens):
        return q4_rows(self.cx, tokens, self.table)

    def step(self, hidden, u, **settings):
        """(tokens, log-probabilities, embedded rows) of the next tick; `settings` as in sample()."""
        tokens, logprob = sample(self.cx, self.logits(hidden), u, **settings)
        return tokens, logprob, self.embed(tokens)
