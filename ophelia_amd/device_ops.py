"""Operators on device tensors over libophelia_seq.so (C ABI: include/ophelia_seq.h), for models that are trained, or that decode
without leaving the GPU.  ophelia_amd.modules offers them beside the host-buffer operators they widen:

  embed_lookup, embed_gradient                    modules.embed     (modules.py:15-44)     with scaling
  gated_recurrence, gated_recurrence_gradient     modules.hc's mix  (modules.py:196-203)   with the previous state as the layer's input
  cross_attention, cross_attention_gradient       networks.Attention (networks.py:286-325) without the monotonic window

Arguments are torch tensors on one GPU: float32, bfloat16 or float16, time-major views and other strides welcome (the last axis is
copied together if it is strided itself).  Calls queue kernels on torch's current stream of that GPU and return new tensors; they never
synchronise, so they can be captured into a graph.  Sums, statistics and states are float32, and no result depends on the order in
which workgroups run.  Gradients are functions of their own: nothing here records for torch's autograd, and tensors that
require gradients are refused outside torch.no_grad().  Bad arguments raise ValueError before anything is queued; there is
no CPU fallback."""
import ctypes as C
import math

from . import _lib

_T = {}


def _torch():
    import torch
    if not _T:
        _T.update({torch.float32: _lib.SEQ_F32, torch.bfloat16: _lib.SEQ_BF16, torch.float16: _lib.SEQ_F16})
    return torch


def _chk(rc):
    if rc < 0:
        raise _lib.OpheliaHipError("libophelia_seq error %d: %s" % (rc, _lib.load_seq().oph_seq_last_error().decode()))
    return rc


def _need(ok, text, *args):
    if not ok:
        raise ValueError(text % args)


def _first(torch, name, t):
    """Checks the tensor that decides type and device of a call."""
    _need(isinstance(t, torch.Tensor) and t.dtype in _T, "%s must be a float32, bfloat16 or float16 tensor", name)
    _need(t.is_cuda, "%s is on %s: the operators run on a GPU only", name, t.device)
    return t.dtype, t.device


def _like(torch, name, t, dtype, device, shape):
    """A tensor of the call: type, device and shape as given (None: any length), unit stride in the last axis."""
    _need(isinstance(t, torch.Tensor) and t.dtype == dtype, "%s must be a %s tensor", name, dtype)
    _need(t.device == device, "%s is on %s, the call on %s", name, t.device, device)
    _need(tuple(t.shape) == tuple(shape), "%s has shape %s, expected %s", name, tuple(t.shape), tuple(shape))
    _need(not (t.requires_grad and torch.is_grad_enabled()), "%s requires a gradient: call under torch.no_grad() and use the gradient function", name)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _lens(torch, name, t, device, B):
    if t is None:
        return None
    _need(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.device == device and tuple(t.shape) == (B,),
          "%s must be an int32 tensor of shape (%d,) on %s", name, B, device)
    return t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(torch, device):
    return torch.cuda.current_stream(device).cuda_stream


def _workspace(torch, nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _strides(field, t, n):
    s = t.stride()
    for i in range(n):
        field[i] = s[i]


# ---- embedding ------------------------------------------------------------------------------------------------------------------
def _ids(torch, ids, device):
    _need(isinstance(ids, torch.Tensor) and ids.dtype in (torch.int32, torch.int64) and ids.device == device,
          "ids must be an int32 or int64 tensor on %s", device)
    return ids.contiguous(), 4 if ids.dtype == torch.int32 else 8


def embed_lookup(ids, table, scale=1.0, zero_pad=True):
    """scale * table[ids]: ids of any shape, table (vocab, units) -> ids.shape + (units,).  zero_pad: id 0 reads as zeros, as
    everywhere in the reference (modules.py:38-40).  An id outside the table reads as zeros."""
    torch = _torch()
    dtype, device = _first(torch, "table", table)
    _need(table.dim() == 2 and table.shape[0] > 0 and table.shape[1] > 0, "table must have two axes, has shape %s", tuple(table.shape))
    table = _like(torch, "table", table, dtype, device, table.shape)
    ids, width = _ids(torch, ids, device)
    V, U = table.shape
    out = torch.empty(tuple(ids.shape) + (U,), dtype=dtype, device=device)
    _chk(_lib.load_seq().oph_seq_embed_lookup(_ptr(ids), width, ids.numel(), _ptr(table), table.stride(0), V, U, float(scale),
                                              int(zero_pad), _T[dtype], _ptr(out), device.index, _stream(torch, device)))
    return out


def embed_gradient(ids, dout, vocab, scale=1.0, zero_pad=True):
    """Gradient of embed_lookup with respect to its table: dout of shape ids.shape + (units,) -> (vocab, units) of dout's type, row v =
    scale * the sum of the dout rows whose id is v, taken in float32 in a fixed order.  Rows that no id names, ids outside the table and,
    with zero_pad, row 0 get zeros / are left out."""
    torch = _torch()
    dtype, device = _first(torch, "dout", dout)
    ids, width = _ids(torch, ids, device)
    _need(dout.dim() >= 1 and dout.shape[-1] > 0, "dout must have a last axis of units, has shape %s", tuple(dout.shape))
    U = dout.shape[-1]
    dout = _like(torch, "dout", dout, dtype, device, tuple(ids.shape) + (U,)).reshape(-1, U)
    _need(isinstance(vocab, int) and vocab > 0, "vocab must be a positive number of rows, is %r", vocab)
    lib = _lib.load_seq()
    ws = _workspace(torch, _chk(lib.oph_seq_embed_workspace(ids.numel(), vocab, U)), device)
    grad = torch.empty((vocab, U), dtype=dtype, device=device)
    _chk(lib.oph_seq_embed_gradient(_ptr(ids), width, ids.numel(), _ptr(dout), dout.stride(0), vocab, U, float(scale), int(zero_pad),
                                    _T[dtype], _ptr(grad), _ptr(ws), ws.numel(), device.index, _stream(torch, device)))
    return grad


# ---- gated linear recurrence -----------------------------------------------------------------------------------------------------
def _recur(torch, x, gate, h0, lengths):
    dtype, device = _first(torch, "x", x)
    _need(x.dim() == 3 and x.shape[2] > 0, "x must be (batch, time, channels), has shape %s", tuple(x.shape))
    B, T, Ch = x.shape
    x = _like(torch, "x", x, dtype, device, (B, T, Ch))
    gate = _like(torch, "gate", gate, dtype, device, (B, T, Ch))
    if h0 is not None:
        h0 = _like(torch, "h0", h0, torch.float32, device, (B, Ch)).contiguous()
    lens = _lens(torch, "lengths", lengths, device, B)
    a = _lib.OphSeqRecur()
    a.x, a.gate, a.h0, a.lens = _ptr(x), _ptr(gate), _ptr(h0), _ptr(lens)
    _strides(a.x_stride, x, 2)
    _strides(a.gate_stride, gate, 2)
    a.B, a.T, a.C, a.dtype = B, T, Ch, _T[dtype]
    return a, dtype, device, (x, gate, h0, lens)


def gated_recurrence(x, gate, h0=None, lengths=None):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t with a = sigmoid(gate): x, gate (B, T, C), h0 (B, C) float32 or None (zeros).  Returns h (B, T, C)
    of x's type and the state after the last step, (B, C) float32, which the next call takes as h0 (T = 1: one decoder step).
    lengths (B) int32: steps at or past a sequence's length are not read, keep its state and have h = 0."""
    torch = _torch()
    a, dtype, device, keep = _recur(torch, x, gate, h0, lengths)
    h = torch.empty((a.B, a.T, a.C), dtype=dtype, device=device)
    last = torch.empty((a.B, a.C), dtype=torch.float32, device=device)
    a.h, a.h_last = _ptr(h), _ptr(last)
    lib = _lib.load_seq()
    ws = _workspace(torch, _chk(lib.oph_seq_recur_workspace(C.byref(a), 0)), device)
    if ws is not None:
        a.workspace, a.workspace_bytes = _ptr(ws), ws.numel()
    _chk(lib.oph_seq_recur_forward(C.byref(a), device.index, _stream(torch, device)))
    return h, last


def gated_recurrence_gradient(dh, x, gate, h, h0=None, dh_last=None, lengths=None):
    """Gradient of gated_recurrence: dh (B, T, C) and dh_last (B, C) float32 or None are the gradients of its two results, h its first
    result.  Returns dx, dgate (B, T, C) and dh0 (B, C) float32; all three are 0 past a sequence's length (dh0 = dh_last for length 0)."""
    torch = _torch()
    a, dtype, device, keep = _recur(torch, x, gate, h0, lengths)
    shape = (a.B, a.T, a.C)
    dh, h = _like(torch, "dh", dh, dtype, device, shape), _like(torch, "h", h, dtype, device, shape)
    if dh_last is not None:
        dh_last = _like(torch, "dh_last", dh_last, torch.float32, device, shape[::2]).contiguous()
    dx, dgate = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
    dh0 = torch.empty(shape[::2], dtype=torch.float32, device=device)
    a.h, a.dh, a.dh_last, a.dx, a.dgate, a.dh0 = _ptr(h), _ptr(dh), _ptr(dh_last), _ptr(dx), _ptr(dgate), _ptr(dh0)
    _strides(a.h_stride, h, 2)
    _strides(a.dh_stride, dh, 2)
    lib = _lib.load_seq()
    ws = _workspace(torch, _chk(lib.oph_seq_recur_workspace(C.byref(a), 1)), device)
    if ws is not None:
        a.workspace, a.workspace_bytes = _ptr(ws), ws.numel()
    _chk(lib.oph_seq_recur_gradient(C.byref(a), device.index, _stream(torch, device)))
    return dx, dgate, dh0


# ---- cross attention ---------------------------------------------------------------------------------------------------------------
def _attention(torch, q, k, v, q_lens, k_lens, key_mask, scale):
    dtype, device = _first(torch, "q", q)
    _need(q.dim() == 4, "q must be (batch, time, heads, head size), has shape %s", tuple(q.shape))
    _need(isinstance(k, torch.Tensor) and k.dim() == 4, "k must be (batch, time, heads, head size)")
    B, Tq, Hq, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    q = _like(torch, "q", q, dtype, device, (B, Tq, Hq, D))
    k = _like(torch, "k", k, dtype, device, (B, Tk, Hk, D))
    v = _like(torch, "v", v, dtype, device, (B, Tk, Hk, D))
    ql, kl = _lens(torch, "q_lens", q_lens, device, B), _lens(torch, "k_lens", k_lens, device, B)
    a = _lib.OphSeqAttn()
    if key_mask is not None:
        _need(isinstance(key_mask, torch.Tensor) and key_mask.dtype in (torch.bool, torch.uint8) and key_mask.device == device and
              tuple(key_mask.shape) == (B, Tk), "key_mask must be a bool tensor of shape (%d, %d) on %s", B, Tk, device)
        a.mask = _ptr(key_mask)
        _strides(a.mask_stride, key_mask, 2)
    a.q, a.k, a.v, a.q_lens, a.k_lens = _ptr(q), _ptr(k), _ptr(v), _ptr(ql), _ptr(kl)
    _strides(a.q_stride, q, 3)
    _strides(a.k_stride, k, 3)
    _strides(a.v_stride, v, 3)
    a.B, a.Tq, a.Tk, a.Hq, a.Hk, a.D, a.dtype = B, Tq, Tk, Hq, Hk, D, _T[dtype]
    a.scale = 1.0 / math.sqrt(D) if scale is None and D else float(scale or 0.0)
    return a, dtype, device, (q, k, v, ql, kl)


def cross_attention(q, k, v, q_lens=None, k_lens=None, key_mask=None, scale=None):
    """Attention of q (B, Tq, Hq, D) over the encoder states k, v (B, Tk, Hk, D): softmax(scale * q k^T) v, scale = D ** -0.5 by default.
    Hq is a multiple of Hk (consecutive query heads share a key head), D a multiple of 8 up to 256, Tq = 1 a decoder step.
    k_lens (B) int32 and key_mask (B, Tk) bool say which keys may be attended, q_lens (B) int32 which queries there are; what is
    excluded is never used, NaN included.  Returns out (B, Tq, Hq, D) and lse (B, Hq, Tq) float32, the logarithm of each row's sum of
    exponentials: exp(scale * q k^T - lse) are the alignments.  A row without key or query has out = 0 and lse = -inf."""
    torch = _torch()
    a, dtype, device, keep = _attention(torch, q, k, v, q_lens, k_lens, key_mask, scale)
    lib = _lib.load_seq()
    nbytes = _chk(lib.oph_seq_attn_workspace(C.byref(a), 0))
    out = torch.empty((a.B, a.Tq, a.Hq, a.D), dtype=dtype, device=device)
    lse = torch.empty((a.B, a.Hq, a.Tq), dtype=torch.float32, device=device)
    ws = _workspace(torch, nbytes, device)
    a.out, a.lse = _ptr(out), _ptr(lse)
    if ws is not None:
        a.workspace, a.workspace_bytes = _ptr(ws), ws.numel()
    _chk(lib.oph_seq_attn_forward(C.byref(a), device.index, _stream(torch, device)))
    return out, lse


def cross_attention_gradient(dout, q, k, v, out, lse, q_lens=None, k_lens=None, key_mask=None, scale=None):
    """Gradient of cross_attention: dout is the gradient of its first result, out and lse what it returned, the rest its arguments.
    Returns dq, dk, dv in the shapes of q, k, v, zero for queries and keys that took no part; k and v heads shared by several query
    heads get the sum over them, expanded (broadcast) inputs the gradient of every copy."""
    torch = _torch()
    a, dtype, device, keep = _attention(torch, q, k, v, q_lens, k_lens, key_mask, scale)
    shape = (a.B, a.Tq, a.Hq, a.D)
    dout = _like(torch, "dout", dout, dtype, device, shape)
    out = _like(torch, "out", out, dtype, device, shape).contiguous()
    lse = _like(torch, "lse", lse, torch.float32, device, (a.B, a.Hq, a.Tq)).contiguous()
    lib = _lib.load_seq()
    nbytes = _chk(lib.oph_seq_attn_workspace(C.byref(a), 1))
    dq = torch.empty(shape, dtype=dtype, device=device)
    dk, dv = (torch.empty((a.B, a.Tk, a.Hk, a.D), dtype=dtype, device=device) for _ in range(2))
    ws = _workspace(torch, nbytes, device)
    a.out, a.lse, a.dout, a.dq, a.dk, a.dv = _ptr(out), _ptr(lse), _ptr(dout), _ptr(dq), _ptr(dk), _ptr(dv)
    _strides(a.dout_stride, dout, 3)
    if ws is not None:
        a.workspace, a.workspace_bytes = _ptr(ws), ws.numel()
    _chk(lib.oph_seq_attn_gradient(C.byref(a), device.index, _stream(torch, device)))
    return dq, dk, dv
