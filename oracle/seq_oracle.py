"""64-bit CPU definitions of the device operators (include/ophelia_seq.h), each with a bound on what a kernel may be off by.

Bounds count roundings.  u = half a step of the result's type (finfo.eps / 2); e = 2^-24, half a step of the float32 the kernels
calculate in.  A float32 sum of n products is off by at most (n + 1) e times the sum of their absolute values, whatever its order;
exp2 / log2 / reciprocal of the hardware are off by at most one step, and their arguments by a relative e each for scaling and
subtraction.  Products of bounds are dropped and covered by the factor SLACK."""
import math

import torch

E = 2.0 ** -24
SLACK = 1.25
F64 = torch.float64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def narrow(dtype):
    """The rounding of probabilities and score gradients to the operand type of the matrix instructions; float32 is not rounded."""
    return 0.0 if dtype == torch.float32 else half_step(dtype)


def valid(lens, B, n):
    if lens is None:
        return torch.ones(B, n, dtype=torch.bool)
    return torch.arange(n)[None, :] < lens.clamp(0, n)[:, None]


def _prep(q, k, v, q_lens, k_lens, key_mask):
    B, Tq, Hq, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    rows, keys = valid(q_lens, B, Tq), valid(k_lens, B, Tk)
    if key_mask is not None:
        keys = keys & (key_mask != 0)
    zero = torch.zeros((), dtype=F64)
    Q = torch.where(rows[:, :, None, None], q.to(F64), zero).transpose(1, 2)
    K = torch.where(keys[:, :, None, None], k.to(F64), zero).transpose(1, 2).repeat_interleave(Hq // Hk, 1)
    V = torch.where(keys[:, :, None, None], v.to(F64), zero).transpose(1, 2).repeat_interleave(Hq // Hk, 1)
    return Q, K, V, rows, keys


def attention(q, k, v, q_lens=None, k_lens=None, key_mask=None, scale=None):
    """out, lse and a dict of what the gradient and the bounds need; (B, H, T, ...) inside."""
    D, Tk = q.shape[3], k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    Q, K, V, rows, keys = _prep(q, k, v, q_lens, k_lens, key_mask)
    ok = rows[:, None, :, None] & keys[:, None, None, :]
    S = torch.where(ok, Q @ K.transpose(2, 3) * scale, torch.tensor(-math.inf, dtype=F64))
    lse = torch.logsumexp(S, 3) if Tk else torch.full(S.shape[:3], -math.inf, dtype=F64)
    P = torch.where(ok, torch.exp(S - torch.where(torch.isinf(lse), 0.0, lse)[..., None]), torch.zeros((), dtype=F64))
    out = P @ V
    u, n = half_step(q.dtype), narrow(q.dtype)
    # a score: its product sum, then scaling, subtraction of the maximum and exp2 on arguments of its size, twice (numerator, sum)
    ds = (D + 3) * E * scale * (Q.abs() @ K.abs().transpose(2, 3))
    top = ds.amax(3) if Tk else torch.zeros_like(lse)
    big = torch.where(ok, S.abs(), torch.zeros_like(S)).amax(3) if Tk else torch.zeros_like(lse)
    rel = 2 * (top + 4 * E * (big + 1)) + (Tk + 40) * E                # of a normalised probability
    A = P @ V.abs()
    out_bound = SLACK * (u * out.abs() + (n + rel[..., None]) * A) + 1e-30
    lse_bound = SLACK * (top + 4 * E * (big + 1) + (Tk + 40) * E + 2 * E * lse.abs())
    if q.dtype == torch.float16:       # below 2^-14 a half step is 2^-25, of the result and of every probability (taken relative to the
        out_bound = out_bound + 2.0 ** -25 * (1 + V.abs().sum(2, keepdim=True))          # largest: their sum is at least 1)
    ctx = dict(Q=Q, K=K, V=V, rows=rows, keys=keys, ok=ok, P=P, rel=rel, scale=scale, out=out, out_bound=out_bound, dtype=q.dtype,
               G=q.shape[2] // k.shape[2])
    return out.transpose(1, 2), lse, out_bound.transpose(1, 2), lse_bound, ctx


def attention_gradient(dout, ctx):
    """dq, dk, dv and their bounds, for a kernel that is handed the out and lse that the forward's bounds admit."""
    Q, K, V, P, scale, G = ctx["Q"], ctx["K"], ctx["V"], ctx["P"], ctx["scale"], ctx["G"]
    dO = torch.where(ctx["rows"][:, :, None, None], dout.to(F64), torch.zeros((), dtype=F64)).transpose(1, 2)
    D, u, n = Q.shape[3], half_step(ctx["dtype"]), narrow(ctx["dtype"])
    dP = dO @ V.transpose(2, 3)
    delta = (dO * ctx["out"]).sum(3, keepdim=True)
    dS = P * (dP - delta) * scale
    dq, dk, dv = dS @ K, dS.transpose(2, 3) @ Q, P.transpose(2, 3) @ dO
    # a score's gradient: P (from lse: both their errors), dP, delta (sum and the error of out), then its rounding
    delta_bound = (dO.abs() * ctx["out_bound"]).sum(3, keepdim=True) + (D + 2) * E * (dO.abs() * ctx["out"].abs()).sum(3, keepdim=True)
    dP_bound = (D + 2) * E * (dO.abs() @ V.abs().transpose(2, 3))
    relp = 2 * ctx["rel"][..., None]
    dS_bound = P * scale * (dP_bound + delta_bound) + (relp + n + 4 * E) * dS.abs() + 2 * E * P * scale * (dP.abs() + delta.abs())
    nk, nq = P.shape[3], P.shape[2] * G
    f16 = 2.0 ** -25 if ctx["dtype"] == torch.float16 else 0.0

    def group(x):
        B, H, T, D_ = x.shape
        return x.reshape(B, H // G, G, T, D_).sum(2)

    # float16: a score's gradient is held in multiples of 2^-25 as long as all of its row's (dq) lie below 2^15, and what bounds those of its
    # key (dk); above, the multiples grow with the largest, from 2^14 on
    wide_q, wide_k = torch.ones(()), torch.ones(())
    if f16 and nk and nq:
        wide_q = ((dS / scale).abs().amax(3, keepdim=True) / 2 ** 14).clamp_min(1)
        most = lambda x: x.reshape(x.shape[0], -1, G).amax(2)[..., None]                  # over a group's heads: (B, Hk, 1)
        wide_k = ((most(dO.norm(dim=3).amax(2)) * V[:, ::G].norm(dim=3) + most(delta.abs().amax((2, 3)))) / 2 ** 14).clamp_min(1)[..., None]
    bq = SLACK * (u * dq.abs() + dS_bound @ K.abs() + (nk + 20) * E * (dS.abs() @ K.abs())) + f16 * (1 + wide_q * scale * K.abs().sum(2, keepdim=True))
    bk = SLACK * (u * group(dk).abs() + group(dS_bound.transpose(2, 3) @ Q.abs()) + (nq + 20) * E * group(dS.abs().transpose(2, 3) @ Q.abs()))
    bv = SLACK * (u * group(dv).abs() + group(((relp + n) * P).transpose(2, 3) @ dO.abs()) + (nq + 20) * E * group(P.transpose(2, 3) @ dO.abs()))
    bk, bv = bk + f16 * (1 + wide_k * scale * group(Q.abs().sum(2, keepdim=True))), bv + f16 * (1 + group(dO.abs().sum(2, keepdim=True)))
    t = lambda x: x.transpose(1, 2)
    return (t(dq), t(group(dk)), t(group(dv))), (t(bq) + 1e-30, t(bk) + 1e-30, t(bv) + 1e-30)


def embed(ids, table, scale=1.0, zero_pad=True):
    V = table.shape[0]
    ok = (ids >= 0) & (ids < V) & ~((ids == 0) & zero_pad)
    rows = table.to(F64)[torch.where(ok, ids, 0).long()] * float(torch.tensor(scale, dtype=torch.float32))
    out = torch.where(ok[..., None], rows, torch.zeros((), dtype=F64))
    return out, (half_step(table.dtype) + E) * out.abs() + (2.0 ** -25 if table.dtype == torch.float16 else 1e-40)


def embed_gradient(ids, dout, vocab, scale=1.0, zero_pad=True):
    U = dout.shape[-1]
    s = float(torch.tensor(scale, dtype=torch.float32))
    i, d = ids.reshape(-1).long(), dout.reshape(-1, U).to(F64)
    ok = (i >= 0) & (i < vocab) & ~((i == 0) & zero_pad)
    i, d = i[ok], d[ok]
    grad, size, count = torch.zeros(vocab, U, dtype=F64), torch.zeros(vocab, U, dtype=F64), torch.zeros(vocab, dtype=F64)
    grad.index_add_(0, i, d)
    size.index_add_(0, i, d.abs())
    count.index_add_(0, i, torch.ones_like(i, dtype=F64))
    grad, size = grad * s, size * abs(s)
    return grad, SLACK * (half_step(dout.dtype) * grad.abs() + (count[:, None] + 2) * E * size) + (2.0 ** -25 if dout.dtype == torch.float16 else 1e-40)


def recurrence(x, gate, h0=None, lengths=None):
    """h, last and their bounds, ctx.  The error of a state: every gate is off by a relative e * (12 + |gate|) (exp2 and its argument,
    reciprocal, product), and a contribution k steps back carries k of them plus the roundings of at most 16 + k steps that combine
    it: n counts them along the recurrence of absolute values m."""
    B, T, C = x.shape
    live = valid(lengths, B, T)[:, :, None]
    z = torch.zeros((), dtype=F64)
    X, g = torch.where(live, x.to(F64), z), torch.where(live, gate.to(F64), z)
    a, keep = torch.sigmoid(g), torch.sigmoid(-g)
    h = torch.zeros(B, T + 1, C, dtype=F64)
    m, n = torch.zeros(B, T + 1, C, dtype=F64), torch.zeros(B, T + 1, C, dtype=F64)
    if h0 is not None:
        h[:, 0] = h0.to(F64)
        m[:, 0] = h[:, 0].abs()
    per = (E * (12 + g.abs().amax())) if T else E
    for t in range(T):
        on = live[:, t]
        h[:, t + 1] = torch.where(on, a[:, t] * h[:, t] + keep[:, t] * X[:, t], h[:, t])
        new = keep[:, t] * X[:, t].abs()
        m[:, t + 1] = torch.where(on, a[:, t] * m[:, t] + new, m[:, t])
        n[:, t + 1] = torch.where(on, a[:, t] * (n[:, t] + m[:, t]) + new, n[:, t])
    state_bound = SLACK * per * (2 * n + 16 * m)
    out = torch.where(live, h[:, 1:], z)
    u = half_step(x.dtype)
    out_bound = torch.where(live, u * h[:, 1:].abs() + state_bound[:, 1:], z) + (2.0 ** -25 if x.dtype == torch.float16 else 1e-38)
    ctx = dict(X=X, a=a, keep=keep, h=h, live=live, per=per, state_bound=state_bound, u=u, dtype=x.dtype)
    return (out, h[:, T].clone()), (out_bound, state_bound[:, T] + 1e-38), ctx


def recurrence_gradient(dh, dh_last, ctx):
    X, a, keep, h, live, per, u = (ctx[k] for k in ("X", "a", "keep", "h", "live", "per", "u"))
    B, T, C = X.shape
    z = torch.zeros((), dtype=F64)
    d = torch.where(live, dh.to(F64), z)
    m = torch.zeros(B, C, dtype=F64) if dh_last is None else dh_last.to(F64).clone()
    big, cnt = m.abs(), torch.zeros_like(m)
    dx, dg, bx, bg = (torch.zeros(B, T, C, dtype=F64) for _ in range(4))
    tiny = 2.0 ** -25 if ctx["dtype"] == torch.float16 else 1e-38
    for t in range(T - 1, -1, -1):
        on = live[:, t]
        l, lm = m + d[:, t], big + d[:, t].abs()
        lb = SLACK * per * (2 * cnt + 16 * lm)
        diff = h[:, t] - X[:, t]
        hb = ctx["state_bound"][:, t] + tiny                        # the float32 state, whatever the forward's result was rounded to
        dx[:, t] = torch.where(on, keep[:, t] * l, z)
        dg[:, t] = torch.where(on, a[:, t] * keep[:, t] * diff * l, z)
        bx[:, t] = torch.where(on, keep[:, t] * lb + u * dx[:, t].abs() + per * dx[:, t].abs(), z) + tiny
        bg[:, t] = torch.where(on, a[:, t] * keep[:, t] * (diff.abs() * lb + hb * lm + per * 2 * diff.abs() * lm) + u * dg[:, t].abs(), z) * SLACK + tiny
        m, big, cnt = torch.where(on, a[:, t] * l, m), torch.where(on, a[:, t] * lm, big), torch.where(on, a[:, t] * (cnt + lm), cnt)
    return (dx, dg, m), (bx, bg, SLACK * per * (2 * cnt + 16 * big) + 1e-38)
