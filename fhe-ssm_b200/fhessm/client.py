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
``FheError``; nothing is converted or copied silently, and no gradient is dropped: an operand that
requires one is refused unless gradients are off.
"""
import ctypes as C
import operator
import struct

import numpy as np
import torch

from . import FheError, _check, lib

_VP = C.c_void_p
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_LEGACY_STREAM = 1      # cudaStreamLegacy: torch calls its default stream 0, which the C-ABI takes for the context's
MAX_VOCAB = 1 << 20
MAX_ROWS = 1 << 30
MAX_COLS = 1 << 20

# fhe_q4 and fhe_sample_cfg as the bytes that the C-ABI reads (packed in 0.4 us; a ctypes structure takes 1.2)
_Q4 = struct.Struct("@PPiiiiqq")
_SAMPLE = struct.Struct("@PPPPfiff")

_fns = None


def _sigs():
    global _fns
    if _fns is None:
        h = lib()
        for name, args in [
            ("fhe_q4_matvec", [_VP, C.c_char_p, _VP, C.c_int, C.c_longlong, C.c_int, _VP, C.c_int, C.c_longlong, _VP]),
            ("fhe_q4_rows", [_VP, C.c_char_p, _VP, C.c_int, _VP, C.c_int, C.c_longlong, _VP]),
            ("fhe_sample", [_VP, C.c_char_p, _VP, C.c_int, C.c_longlong, C.c_int, C.c_int, _VP, _VP, _VP, _VP]),
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
    if not t.is_cuda or t.get_device() != device:
        raise _bad(f"{what} is not on the context's GPU (cuda:{device})")


def _no_gradient(*named):
    # nothing here is differentiable: a gradient that somebody waits for is refused, not dropped
    if torch.is_grad_enabled():
        for t, what in named:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise _bad(f"{what} requires a gradient, which this call does not have: detach it, or call under torch.no_grad()")


def _rows_of(t, what):
    """(type, row count, row length, row stride) of a 2-d tensor with contiguous rows."""
    shape = t.shape
    if len(shape) != 2:
        raise _bad(f"{what}: expected rows x columns, got {tuple(shape)}")
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise _bad(f"{what}: float32, float16 or bfloat16, got {t.dtype}")
    m, n = shape
    if t.is_contiguous():
        return kind, m, n, n
    ld, step = t.stride()
    if n > 1 and step != 1:
        raise _bad(f"{what}: the values of a row are not contiguous")
    if m > 1 and ld < n:
        raise _bad(f"{what}: rows overlap")
    return kind, m, n, ld if m > 1 else n


def _whole(what, *values):
    try:
        return [operator.index(v) for v in values]
    except TypeError:
        raise _bad(f"{what}: columns and group are whole numbers") from None


class Q4Table:
    """A table of rows x cols values in 4 bits with a scale for each `group` columns of a row:
    value (i, c) = scale[i, c // group] * (q - 8), q the low (even c) or high (odd c) half of byte
    weight[i, c // 2].  weight: uint8 (rows, bytes), a row padded to a multiple of 16 bytes;
    scale: float32, float16 or bfloat16 (rows, ceil(cols / group)); group: a multiple of 32."""

    __slots__ = ("weight", "scale", "rows", "cols", "group", "device", "c")

    def __init__(self, weight, scale, *, cols, group):
        if weight.dtype != torch.uint8 or weight.dim() != 2:
            raise _bad("q4 table: weight is a uint8 tensor, rows x bytes")
        rows, nbytes = weight.shape
        cols, group = _whole("q4 table", cols, group)
        if not 1 <= cols <= MAX_COLS or group < 32 or group % 32 or group >= 1 << 31:
            raise _bad(f"q4 table: 1 to {MAX_COLS} columns and a group that is a multiple of 32")
        if rows > MAX_ROWS:
            raise _bad(f"q4 table: {MAX_ROWS} rows at most")
        if nbytes < -(-cols // 32) * 16:
            raise _bad("q4 table: rows are padded to a multiple of 16 bytes (32 columns)")
        st, srows, groups, lds = _rows_of(scale, "q4 scales")
        if srows != rows or groups != -(-cols // group):
            raise _bad(f"q4 scales: expected {(rows, -(-cols // group))}, got {tuple(scale.shape)}")
        self.device = weight.get_device()
        if scale.get_device() != self.device:
            raise _bad("q4 table: weight and scale are on different devices")
        ldq = nbytes
        if not weight.is_contiguous():
            ldq, step = weight.stride()
            if step != 1 or (rows > 1 and ldq < nbytes):
                raise _bad("q4 table: the bytes of a row are not contiguous, or rows overlap")
        if rows <= 1:
            ldq = -(-nbytes // 16) * 16
        self.weight, self.scale, self.rows, self.cols, self.group = weight, scale, rows, cols, group
        self.c = _Q4.pack(weight.data_ptr(), scale.data_ptr(), st, rows, cols, group, ldq, lds)

    @classmethod
    def quantise(cls, w, *, group=64, scale_dtype=torch.float16, device="cpu"):
        """The 4-bit table nearest to w (rows x cols, a float array or tensor): a group's scale is its largest
        magnitude over 7, rounded to scale_dtype."""
        w = w.detach() if torch.is_tensor(w) else torch.as_tensor(np.asarray(w))
        w = w.to(device=device, dtype=torch.float32)
        group, = _whole("quantise", group)
        if w.dim() != 2 or group < 32 or group % 32:
            raise _bad("quantise: rows x cols and a group that is a multiple of 32")
        if scale_dtype not in _TYPES:
            raise _bad(f"quantise: scales in float32, float16 or bfloat16, not {scale_dtype}")
        rows, cols = w.shape
        groups = -(-cols // group)
        wide = torch.zeros(rows, groups * group, dtype=torch.float32, device=w.device)
        wide[:, :cols] = w
        wide = wide.view(rows, groups, group)
        scale = (wide.abs().amax(2) / 7).to(scale_dtype)
        if not torch.isfinite(scale).all():
            raise _bad(f"quantise: values that are not finite, or too large for a scale in {scale_dtype}")
        s = scale.float().unsqueeze(2)
        q = torch.where(s > 0, torch.round(wide / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(wide))
        q = (q.clamp(-8, 7) + 8).to(torch.uint8).view(rows, groups * group)[:, :-(-cols // 32) * 32]
        return cls((q[:, 0::2] | q[:, 1::2] << 4).contiguous(), scale.contiguous(), cols=cols, group=group)

    def to(self, device):
        return Q4Table(self.weight.to(device), self.scale.to(device), cols=self.cols, group=self.group)

    def dequantise(self):
        """The table's values, float32 (rows, cols)."""
        q = torch.stack([self.weight & 15, self.weight >> 4], dim=-1).flatten(-2)[:, :self.cols].float() - 8
        return q * self.scale.float().repeat_interleave(self.group, dim=1)[:, :self.cols]


def _out(out, like, m, n, dtype, device):
    """(output, its type, its row stride): a new one, or the caller's."""
    kind = _TYPES.get(dtype)
    if kind is None:
        raise _bad(f"out: float32, float16 or bfloat16, got {dtype}")
    if out is None:
        return like.new_empty((m, n), dtype=dtype), kind, n
    if tuple(out.shape) != (m, n) or out.dtype != dtype:
        raise _bad(f"out: expected {dtype} {(m, n)}, got {out.dtype} {tuple(out.shape)}")
    _on_gpu(device, out, "out")
    return out, kind, _rows_of(out, "out")[3]


def q4_matvec(cx, x, table, *, dtype=torch.float32, out=None):
    """x (m, cols) times the table's transpose: (m, rows) of `dtype` (fhe_q4_matvec).  x: float32,
    float16 or bfloat16 with contiguous rows (any row stride), 2^21 of them at most.  Two float32 rows at a time are
    held whole; of more, on most tables, a value is held to 22 bits and to 2^-39 of its row's largest.  A kernel whose
    bounded wait runs out leaves NaN, and ``cx.sync()`` raises once the stream is synchronised."""
    xt, m, k, ldx = _rows_of(x, "x")
    _no_gradient((x, "x"), (table.scale, "the table's scale"), (out, "out"))
    if k != table.cols:
        raise _bad(f"x has {k} columns, the table {table.cols}")
    device = cx.p.device
    _on_gpu(device, x, "x")
    if table.device != device:
        raise _bad(f"q4 table is not on the context's GPU (cuda:{device})")
    out, ot, ldo = _out(out, x, m, table.rows, dtype, device)
    _check((_fns or _sigs()).fhe_q4_matvec(cx.h, table.c, x.data_ptr(), xt, ldx, m, out.data_ptr(), ot, ldo,
                                           _stream(device)))
    return out


def q4_rows(cx, tokens, table, *, dtype=torch.float32, out=None):
    """Rows of the table by token id: tokens (m,) int64 -> (m, cols) of `dtype` (fhe_q4_rows); a token
    outside the table (the -1 of an empty row) gives zeros."""
    if tokens.dim() != 1 or tokens.dtype != torch.int64 or not tokens.is_contiguous():
        raise _bad("tokens: a contiguous int64 vector")
    _no_gradient((table.scale, "the table's scale"), (out, "out"))
    device = cx.p.device
    _on_gpu(device, tokens, "tokens")
    if table.device != device:
        raise _bad(f"q4 table is not on the context's GPU (cuda:{device})")
    m = tokens.shape[0]
    out, ot, ldo = _out(out, tokens, m, table.cols, dtype, device)
    _check((_fns or _sigs()).fhe_q4_rows(cx.h, table.c, tokens.data_ptr(), m, out.data_ptr(), ot, ldo,
                                         _stream(device)))
    return out


def _setting(device, v, rows, dtype, what):
    """(device pointer or 0, plain value) of a setting given as one number or as a value per row."""
    if not isinstance(v, torch.Tensor):
        return 0, v
    if v.dim() != 1 or v.shape[0] != rows or v.dtype != dtype or not v.is_contiguous():
        raise _bad(f"{what}: one number, or a contiguous {dtype} vector with a value for each row")
    _on_gpu(device, v, what)
    return v.data_ptr(), 0


def sample(cx, logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token per row of logits (rows, vocab) from the random numbers u (rows,) in [0, 1): (tokens
    int64, log-probabilities float32) (fhe_sample, whose comment defines the choice).  Each setting is
    one number or a vector with a value for each row (float32; top_k int32).  temperature 0: the
    largest logit.  top_k 0, top_p 1 and min_p 0 are off.  The token of a row that allows none is -1."""
    lt, rows, vocab, ld = _rows_of(logits, "logits")
    _no_gradient((logits, "logits"), (temperature, "temperature"), (top_p, "top_p"), (min_p, "min_p"), (u, "u"))
    device = cx.p.device
    _on_gpu(device, logits, "logits")
    if not 1 <= vocab <= MAX_VOCAB:
        raise _bad(f"logits: a vocabulary of 1 to {MAX_VOCAB}")
    up, _ = _setting(device, u, rows, torch.float32, "u")
    if not isinstance(u, torch.Tensor):
        raise _bad("u: a float32 vector with a random number for each row")
    t, t1 = _setting(device, temperature, rows, torch.float32, "temperature")
    k, k1 = _setting(device, top_k, rows, torch.int32, "top_k")
    p, p1 = _setting(device, top_p, rows, torch.float32, "top_p")
    mp, mp1 = _setting(device, min_p, rows, torch.float32, "min_p")
    token, logprob = u.new_empty(rows, dtype=torch.int64), u.new_empty(rows)
    try:
        cfg = _SAMPLE.pack(t, k, p, mp, t1, k1 if k1 < vocab else vocab, p1, mp1)
    except (struct.error, OverflowError, TypeError) as e:
        raise _bad(f"sample: a setting is not a number of its type ({e})")
    _check((_fns or _sigs()).fhe_sample(cx.h, cfg, logits.data_ptr(), lt, ld, rows, vocab, up, token.data_ptr(),
                                        logprob.data_ptr(), _stream(device)))
    return token, logprob


class TokenHead:
    """The client's side of a decode tick with a tied 4-bit table: decrypted normed rows in, tokens and the
    next tick's input rows out.  Only for a tied table: a model with an embedding of its own (RWKV-7) takes
    q4_matvec with its head's table, after its output norm, and q4_rows with its embedding's, into which its
    input norm is folded."""

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
        """(tokens, log-probabilities, embedded rows) of the next tick; `settings` as in sample().  Logits that were lost
        (q4_matvec's NaN) come out as token -1 and a row of zeros: call ``cx.sync()`` once a tick, when the stream is
        synchronised, which raises for them."""
        tokens, logprob = sample(self.cx, self.logits(hidden), u, **settings)
        return tokens, logprob, self.embed(tokens)
