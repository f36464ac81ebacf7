"""Operators on device tensors over libophelia_seq.so (C ABI: include/ophelia_seq.h), for models that are trained, or that decode
without leaving the GPU.  ophelia_amd.modules offers them beside the host-buffer operators they widen:

  embed_lookup, embed_gradient                    modules.embed     (modules.py:15-44)     with scaling
  gated_recurrence, gated_recurrence_gradient     modules.hc's mix  (modules.py:196-203)   with the previous state as the layer's input
  cross_attention, cross_attention_gradient       networks.Attention (networks.py:286-325) without the monotonic window

Arguments are torch tensors on one GPU: float32, bfloat16 or float16, time-major views and other strides welcome (the last axis is
copied together if it is strided itself).  Calls queue kernels on torch's current stream of that GPU and return new tensors; they never
synchronise, so they can be captured into a graph.  Sums, statistics and states are float32, and no result depends on the order in
which workgroups run.  Gradients are functions of their own: nothing here records for torch's autograd, tensors that require
gradients are refused outside torch.no_grad(), and tensors that carry a forward-mode tangent always.  Bad arguments raise before anything is queued: types, shapes, devices and
sizes beyond 32 bits ValueError, what the library refuses (head sizes and counts, scales, sizes that it does not do) OpheliaHipError.
There is no CPU fallback."""
import ctypes
import operator
import struct

from . import _lib

_T = {}
_torch = None                 # the module, and below the library and the stream's raw handle: found at the first call
_seq = None
_stream = None
_forward = None               # torch.autograd.forward_ad
# the argument structures of include/ophelia_seq.h as the compiler lays them out: packing them in one go is a third of the time that filling
# ctypes fields takes, and a call on small tensors is bound by what happens here
_ATTN = struct.Struct("@12P14qPN7if")
_RECUR = struct.Struct("@11P8qPN4i")


def _setup():
    global _torch, _seq, _stream, _forward
    import torch
    _forward = torch.autograd.forward_ad
    _T.update({torch.float32: _lib.SEQ_F32, torch.bfloat16: _lib.SEQ_BF16, torch.float16: _lib.SEQ_F16})
    # the raw handle of the current stream without the stream object around it, where this torch has it
    _stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
    _seq = _lib.load_seq()
    _torch = torch
    return torch


def _chk(rc):
    if rc < 0:
        raise _lib.OpheliaHipError("libophelia_seq error %d: %s" % (rc, _seq.oph_seq_last_error().decode()))
    return rc


def _first(torch, name, t):
    """Checks the tensor that decides type and device of a call."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _T:
        raise ValueError("%s must be a float32, bfloat16 or float16 tensor" % name)
    if not t.is_cuda:
        raise ValueError("%s is on %s: the operators run on a GPU only" % (name, t.device))
    return t.dtype, t.device


def _like(torch, name, t, dtype, device, shape):
    """A tensor of the call: type, device and shape as given, unit stride in the last axis."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device and not t.requires_grad and _forward._current_level < 0:
        return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise ValueError("%s must be a %s tensor" % (name, dtype))
    if t.device != device:
        raise ValueError("%s is on %s, the call on %s" % (name, t.device, device))
    if t.shape != shape:
        raise ValueError("%s has shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires a gradient: call under torch.no_grad() and use the gradient function" % name)
    if _forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None:      # not a matter of no_grad()
        raise ValueError("%s carries a forward-mode tangent, which would be lost: unpack it first" % name)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _lens(torch, name, t, device, B):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device or t.shape != (B,):
        raise ValueError("%s must be an int32 tensor of shape (%d,) on %s" % (name, B, device))
    return t.contiguous()


def _sizes(what, sizes):
    """The library takes sizes as 32-bit numbers; larger ones (of expanded tensors) must not arrive there as others."""
    if max(sizes) > 2147483647:
        raise ValueError("%s: a size of %d, the largest is 2147483647" % (what, max(sizes)))
    return tuple(sizes)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _workspace(torch, nbytes, device):
    """Scratch memory of one call, from torch's allocator: its next user on this stream comes after the call, a captured graph owns its own."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


# ---- embedding ------------------------------------------------------------------------------------------------------------------
def _ids(torch, ids, device):
    if not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int32, torch.int64) or ids.device != device:
        raise ValueError("ids must be an int32 or int64 tensor on %s" % device)
    return ids.contiguous(), 4 if ids.dtype == torch.int32 else 8


def embed_lookup(ids, table, scale=1.0, zero_pad=True):
    """scale * table[ids]: ids of any shape, table (vocab, units) -> ids.shape + (units,).  zero_pad: id 0 reads as zeros, as
    everywhere in the reference (modules.py:38-40).  An id outside the table reads as zeros."""
    torch = _torch or _setup()
    dtype, device = _first(torch, "table", table)
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError("table must be (vocab, units), has shape %s" % (tuple(table.shape),))
    table = _like(torch, "table", table, dtype, device, table.shape)
    ids, width = _ids(torch, ids, device)
    V, U = _sizes("table", table.shape)
    out = table.new_empty(ids.shape + (U,))
    _chk(_seq.oph_seq_embed_lookup(ids.data_ptr(), width, ids.numel(), table.data_ptr(), table.stride(0), V, U, float(scale),
                                   bool(zero_pad), _T[dtype], out.data_ptr(), device.index, _stream(device.index)))
    return out


def embed_gradient(ids, dout, vocab, scale=1.0, zero_pad=True):
    """Gradient of embed_lookup with respect to its table: dout of shape ids.shape + (units,) -> (vocab, units) of dout's type, row v =
    scale * the sum of the dout rows whose id is v, taken in float32 in a fixed order.  Rows that no id names, and with zero_pad row 0, are
    zeros; ids outside the table are left out."""
    torch = _torch or _setup()
    vocab = operator.index(vocab)
    if vocab < 1 or vocab > 2147483647:
        raise ValueError("vocab must be a number of rows from 1 to 2147483647, is %d" % vocab)
    dtype, device = _first(torch, "dout", dout)
    ids, width = _ids(torch, ids, device)
    if dout.dim() < 1 or dout.shape[-1] < 1:
        raise ValueError("dout must have a last axis of units, has shape %s" % (tuple(dout.shape),))
    U = _sizes("dout", dout.shape[-1:])[0]
    dout = _like(torch, "dout", dout, dtype, device, ids.shape + (U,))
    if dout.dim() != 2:
        dout = dout.reshape(-1, U)
    n = ids.numel()
    nbytes = _chk(_seq.oph_seq_embed_workspace(n, vocab, U))
    ws = _workspace(torch, nbytes, device) if nbytes else None
    grad = dout.new_empty((vocab, U))
    _chk(_seq.oph_seq_embed_gradient(ids.data_ptr(), width, n, dout.data_ptr(), dout.stride(0), vocab, U, float(scale), bool(zero_pad),
                                     _T[dtype], grad.data_ptr(), _ptr(ws), nbytes, device.index, _stream(device.index)))
    return grad


# ---- gated linear recurrence -----------------------------------------------------------------------------------------------------
def _recur(torch, x, gate, h0, lengths):
    dtype, device = _first(torch, "x", x)
    if x.dim() != 3 or x.shape[2] < 1:
        raise ValueError("x must be (batch, time, channels), has shape %s" % (tuple(x.shape),))
    shape = x.shape
    _sizes("x", shape)
    x = _like(torch, "x", x, dtype, device, shape)
    gate = _like(torch, "gate", gate, dtype, device, shape)
    if h0 is not None:
        h0 = _like(torch, "h0", h0, torch.float32, device, (shape[0], shape[2])).contiguous()
    return dtype, device, shape, x, gate, h0, _lens(torch, "lengths", lengths, device, shape[0])


def _run_recur(torch, call, gradient, pointers, strides, shape, dtype, device):
    """Fills the argument structure (include/ophelia_seq.h: oph_seq_recur), finds the workspace and makes the call."""
    sizes = tuple(shape) + (_T[dtype],)
    a = _RECUR.pack(*pointers, *strides, 0, 0, *sizes)
    nbytes = _chk(_seq.oph_seq_recur_workspace(a, gradient))
    if nbytes:
        ws = _workspace(torch, nbytes, device)
        a = _RECUR.pack(*pointers, *strides, ws.data_ptr(), nbytes, *sizes)
    _chk(call(a, device.index, _stream(device.index)))


def gated_recurrence(x, gate, h0=None, lengths=None):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t with a = sigmoid(gate): x, gate (B, T, C), h0 (B, C) float32 or None (zeros).  Returns h (B, T, C)
    of x's type and the state after the last step, (B, C) float32, which the next call takes as h0 (T = 1: one decoder step).
    lengths (B) int32: steps at or past a sequence's length are not read, keep its state and have h = 0."""
    torch = _torch or _setup()
    dtype, device, shape, x, gate, h0, lens = _recur(torch, x, gate, h0, lengths)
    h = x.new_empty(shape)
    last = x.new_empty((shape[0], shape[2]), dtype=torch.float32)
    _run_recur(torch, _seq.oph_seq_recur_forward, 0,
               (x.data_ptr(), gate.data_ptr(), _ptr(h0), h.data_ptr(), last.data_ptr(), 0, 0, 0, 0, 0, _ptr(lens)),
               x.stride()[:2] + gate.stride()[:2] + (0, 0, 0, 0), shape, dtype, device)
    return h, last


def gated_recurrence_gradient(dh, x, gate, h, h0=None, dh_last=None, lengths=None):
    """Gradient of gated_recurrence: dh (B, T, C) and dh_last (B, C) float32 or None are the gradients of its two results, h its first
    result (float32: the states that the gradient needs; in 16 bits it forms them again, unrounded, from x, gate and h0).  Returns dx,
    dgate (B, T, C), 0 past a sequence's length, and dh0 (B, C) float32 (dh_last for a sequence of length 0)."""
    torch = _torch or _setup()
    dtype, device, shape, x, gate, h0, lens = _recur(torch, x, gate, h0, lengths)
    dh, h = _like(torch, "dh", dh, dtype, device, shape), _like(torch, "h", h, dtype, device, shape)
    state = (shape[0], shape[2])
    if dh_last is not None:
        dh_last = _like(torch, "dh_last", dh_last, torch.float32, device, state).contiguous()
    dx, dgate, dh0 = x.new_empty(shape), x.new_empty(shape), x.new_empty(state, dtype=torch.float32)
    _run_recur(torch, _seq.oph_seq_recur_gradient, 1,
               (x.data_ptr(), gate.data_ptr(), _ptr(h0), h.data_ptr(), 0, dh.data_ptr(), _ptr(dh_last), dx.data_ptr(), dgate.data_ptr(),
                dh0.data_ptr(), _ptr(lens)),
               x.stride()[:2] + gate.stride()[:2] + h.stride()[:2] + dh.stride()[:2], shape, dtype, device)
    return dx, dgate, dh0


# ---- cross attention ---------------------------------------------------------------------------------------------------------------
def _attention(torch, q, k, v, q_lens, k_lens, key_mask, scale):
    dtype, device = _first(torch, "q", q)
    if q.dim() != 4:
        raise ValueError("q must be (batch, time, heads, head size), has shape %s" % (tuple(q.shape),))
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("k must be (batch, time, heads, head size)")
    B, Tq, Hq, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    _sizes("q and k", (B, Tq, Tk, Hq, Hk, D))
    shape = (B, Tk, Hk, D)
    q = _like(torch, "q", q, dtype, device, q.shape)
    k, v = _like(torch, "k", k, dtype, device, shape), _like(torch, "v", v, dtype, device, shape)
    ql, kl = _lens(torch, "q_lens", q_lens, device, B), _lens(torch, "k_lens", k_lens, device, B)
    if key_mask is not None and (not isinstance(key_mask, torch.Tensor) or key_mask.dtype not in (torch.bool, torch.uint8) or
                                 key_mask.device != device or key_mask.shape != (B, Tk)):
        raise ValueError("key_mask must be a bool tensor of shape (%d, %d) on %s" % (B, Tk, device))
    # a scale that float32 does not hold is infinite there, which the library refuses
    sizes = (B, Tq, Tk, Hq, Hk, D, _T[dtype], D ** -0.5 if scale is None and D else ctypes.c_float(scale or 0.0).value)
    return dtype, device, q, k, v, ql, kl, sizes


def _run_attention(torch, call, gradient, pointers, strides, sizes, device):
    """Fills the argument structure (include/ophelia_seq.h: oph_seq_attn), finds the workspace and makes the call."""
    a = _ATTN.pack(*pointers, *strides, 0, 0, *sizes)
    nbytes = _chk(_seq.oph_seq_attn_workspace(a, gradient))
    if nbytes:
        ws = _workspace(torch, nbytes, device)
        a = _ATTN.pack(*pointers, *strides, ws.data_ptr(), nbytes, *sizes)
    _chk(call(a, device.index, _stream(device.index)))


def cross_attention(q, k, v, q_lens=None, k_lens=None, key_mask=None, scale=None):
    """Attention of q (B, Tq, Hq, D) over the encoder states k, v (B, Tk, Hk, D): softmax(scale * q k^T) v, scale = D ** -0.5 by default.
    Hq is a multiple of Hk (consecutive query heads share a key head), D a multiple of 8 up to 256, Tq = 1 a decoder step.
    k_lens (B) int32 and key_mask (B, Tk) bool say which keys may be attended, q_lens (B) int32 which queries there are; what is
    excluded is never used, NaN included.  Returns out (B, Tq, Hq, D) and lse (B, Hq, Tq) float32, the logarithm of each row's sum of
    exponentials: exp(scale * q k^T - lse) are the alignments.  A row without key or query has out = 0 and lse = -inf."""
    torch = _torch or _setup()
    dtype, device, q, k, v, ql, kl, sizes = _attention(torch, q, k, v, q_lens, k_lens, key_mask, scale)
    out = q.new_empty(q.shape)
    lse = q.new_empty((sizes[0], sizes[3], sizes[1]), dtype=torch.float32)
    mask = (0, 0) if key_mask is None else key_mask.stride()
    _run_attention(torch, _seq.oph_seq_attn_forward, 0,
                   (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), 0, 0, 0, 0, _ptr(ql), _ptr(kl), _ptr(key_mask)),
                   q.stride()[:3] + k.stride()[:3] + v.stride()[:3] + (0, 0, 0) + mask, sizes, device)
    return out, lse


def cross_attention_gradient(dout, q, k, v, out, lse, q_lens=None, k_lens=None, key_mask=None, scale=None):
    """Gradient of cross_attention: dout is the gradient of its first result, out and lse what it returned, the rest its arguments.
    Returns dq, dk, dv in the shapes of q, k, v, zero for queries and keys that took no part; k and v heads shared by several query
    heads get the sum over them, expanded (broadcast) inputs the gradient of every copy."""
    torch = _torch or _setup()
    dtype, device, q, k, v, ql, kl, sizes = _attention(torch, q, k, v, q_lens, k_lens, key_mask, scale)
    dout = _like(torch, "dout", dout, dtype, device, q.shape)
    out = _like(torch, "out", out, dtype, device, q.shape).contiguous()
    lse = _like(torch, "lse", lse, torch.float32, device, (sizes[0], sizes[3], sizes[1])).contiguous()
    dq, dk, dv = q.new_empty(q.shape), q.new_empty(k.shape), q.new_empty(k.shape)
    mask = (0, 0) if key_mask is None else key_mask.stride()
    _run_attention(torch, _seq.oph_seq_attn_gradient, 1,
                   (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                    dv.data_ptr(), _ptr(ql), _ptr(kl), _ptr(key_mask)),
                   q.stride()[:3] + k.stride()[:3] + v.stride()[:3] + dout.stride()[:3] + mask, sizes, device)
    return dq, dk, dv
