"""GPU parity of the device operators (ophelia_amd.device_ops over libophelia_seq.so) with their 64-bit definitions: every element within
the bound that counting the roundings allows (oracle/seq_oracle.py)."""
import math

import pytest
import torch

from oracle import seq_oracle as O

pytestmark = pytest.mark.gpu
DT = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]
dtypes = pytest.mark.parametrize("dt", DT, ids=IDS)


def _rand(seed, shape, dt, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float32) * scale).to(dt)


def _within(name, got, ref, bound):
    got = got.double().cpu()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    same = (got == ref)                                     # infinities
    off = torch.where(same, torch.zeros_like(ref), (got - ref).abs())
    bad = ~(off <= bound)                                   # NaN is bad
    assert not bad.any(), "%s: %d of %d beyond the bound, worst %.3g times, first at %s: %r instead of %r" % (
        name, int(bad.sum()), bad.numel(), float((off / bound).nan_to_num(math.inf).max()), bad.nonzero()[0].tolist(),
        got[bad][0].item(), ref[bad][0].item())


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


# ---- cross attention ---------------------------------------------------------------------------------------------------------------
# few rows (split keys, one and several splits), many rows (shared tiles), head sizes on and off the kernels' 64 / 128 / 256
SHAPES = [(1, 1, 1, 1, 1, 8), (3, 1, 150, 1, 1, 256), (2, 1, 1000, 8, 2, 128), (2, 5, 333, 6, 3, 64), (2, 67, 129, 6, 2, 40), (1, 200, 150, 1, 1, 256),
          (2, 33, 31, 2, 2, 192), (2, 130, 65, 4, 4, 128), (1, 1, 2100, 4, 1, 64), (3, 2, 0, 2, 1, 16), (8, 260, 70, 16, 16, 24), (4, 130, 97, 96, 32, 72),
          (9, 200, 70, 24, 24, 136), (4, 129, 33, 64, 32, 128)]


def _case(shape, dt, seed):
    B, Tq, Tk, Hq, Hk, D = shape
    return (_rand(seed, (B, Tq, Hq, D), dt), _rand(seed + 1, (B, Tk, Hk, D), dt), _rand(seed + 2, (B, Tk, Hk, D), dt), _rand(seed + 3, (B, Tq, Hq, D), dt))


def _masks(kind, B, Tq, Tk, seed=5):
    """(q_lens, k_lens, key_mask): whole; ragged with an empty sequence and lengths outside the axis; ragged and masked, one row of the
    mask false throughout."""
    if kind == "whole":
        return None, None, None
    g = torch.Generator().manual_seed(seed)
    ql = torch.randint(0, Tq + 1, (B,), generator=g, dtype=torch.int32)
    kl = torch.randint(0, Tk + 1, (B,), generator=g, dtype=torch.int32)
    ql[0], kl[0] = Tq + 3, Tk + 7
    if B > 1:
        kl[1] = -2
    if kind == "ragged":
        return ql, kl, None
    mask = torch.rand(B, Tk, generator=g) < 0.6
    mask[B - 1] = False
    return None, kl, mask


def _attend(shape, dt, kind, seed=11, scale=None, spoil=False):
    from ophelia_amd import modules as M
    B, Tq, Tk, Hq, Hk, D = shape
    q, k, v, do = _case(shape, dt, seed)
    ql, kl, mask = _masks(kind, B, Tq, Tk)
    out, lse, bo, bl, ctx = O.attention(q, k, v, ql, kl, mask, scale)
    if spoil:                                               # what is excluded must not be used, whatever it holds
        rows, keys = ctx["rows"], ctx["keys"]
        q[~rows], do[~rows] = math.nan, math.inf
        k[~keys], v[~keys] = math.inf, math.nan
    dev = dict(zip(("q_lens", "k_lens", "key_mask"), _cuda(ql, kl, mask)), scale=scale)
    qd, kd, vd, dd = _cuda(q, k, v, do)
    o, l = M.cross_attention(qd, kd, vd, **dev)
    _within("out", o, out, bo)
    _within("lse", l, lse, bl)
    ref, bound = O.attention_gradient(torch.where(ctx["rows"][:, :, None, None], do, torch.zeros((), dtype=dt)), ctx)
    if spoil:
        o = o.clone()
        o[~ctx["rows"].cuda()] = math.nan
    got = M.cross_attention_gradient(dd, qd, kd, vd, o, l, **dev)
    for n, g, r, b in zip(("dq", "dk", "dv"), got, ref, bound):
        _within(n, g, r, b)


@dtypes
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(shape, dt):
    _attend(shape, dt, "whole")


@dtypes
@pytest.mark.parametrize("kind", ["ragged", "masked"])
@pytest.mark.parametrize("shape", [(5, 2, 90, 1, 1, 64), (4, 2, 300, 4, 2, 128), (3, 1, 150, 2, 1, 256), (4, 40, 77, 4, 2, 64), (9, 129, 70, 32, 32, 48), (3, 5, 700, 4, 2, 128), (2, 300, 200, 2, 1, 96), (2, 70, 200, 3, 1, 200)], ids=str)
def test_attention_excluded_places_are_never_used(shape, kind, dt):
    _attend(shape, dt, kind, spoil=True)


@dtypes
def test_attention_large_scores_and_own_scale(dt):
    """scores of +-60 (a softmax that is all but one-hot) and a scale that is not D ** -0.5."""
    _attend((2, 70, 90, 2, 1, 64), dt, "whole", scale=2.0)
    _attend((2, 1, 300, 4, 1, 64), dt, "ragged", scale=0.01)


@dtypes
def test_attention_strides_and_odd_alignment(dt):
    """head-major views, keys and values interleaved in one buffer, buffers that start at an odd element: the contiguous call's bits."""
    from ophelia_amd import modules as M
    B, Tq, Tk, Hq, Hk, D = 2, 37, 75, 4, 2, 40
    q, k, v, do = _cuda(*_case((B, Tq, Tk, Hq, Hk, D), dt, 3))
    o, l = M.cross_attention(q, k, v)
    g = M.cross_attention_gradient(do, q, k, v, o, l)

    def odd(t, order):
        buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
        p = t.permute(order).contiguous()
        buf.copy_(p.reshape(-1))
        back = [order.index(i) for i in range(4)]
        return buf.view(p.shape).permute(back)

    kv = torch.zeros(B, Tk, Hk, 2 * D + 3, dtype=dt, device="cuda")
    kv[..., :D], kv[..., D + 3:] = k, v
    q2, do2, k2, v2 = odd(q, (0, 2, 1, 3)), odd(do, (2, 0, 1, 3)), kv[..., :D], kv[..., D + 3:]
    mask = torch.ones(Tk, 2 * B, dtype=torch.bool, device="cuda").t()[::2]
    o2, l2 = M.cross_attention(q2, k2, v2, key_mask=mask)
    assert torch.equal(o, o2) and torch.equal(l, l2)
    for x, y in zip(g, M.cross_attention_gradient(do2, q2, k2, v2, o2, l2, key_mask=mask)):
        assert torch.equal(x, y)
    last = torch.empty(B, Tk, Hk, D, 2, dtype=dt, device="cuda")[..., 0]         # the last axis strided: copied together
    last.copy_(k)
    assert torch.equal(M.cross_attention(q, last, v)[0], o)


def test_attention_broadcast_keys():
    """One encoder state for the whole batch (stride 0): the gradient of every copy, whose sum is the shared state's."""
    from ophelia_amd import modules as M
    q, k, v, do = _case((3, 20, 50, 2, 1, 64), torch.float32, 8)
    k, v = k[:1], v[:1]
    ctx = O.attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1))[4]
    ref, bound = O.attention_gradient(do, ctx)
    qd, kd, vd, dd = _cuda(q, k, v, do)
    ke, ve = kd.expand(3, -1, -1, -1), vd.expand(3, -1, -1, -1)
    o, l = M.cross_attention(qd, ke, ve)
    for n, g, r, b in zip(("dq", "dk", "dv"), M.cross_attention_gradient(dd, qd, ke, ve, o, l), ref, bound):
        _within(n, g, r, b)


@pytest.mark.parametrize("axis", ["batch", "time"])
def test_attention_offsets_beyond_32_bits(axis):
    """keys in a cache whose sequences, or steps, lie more than 2^31 elements apart."""
    from ophelia_amd import modules as M
    B, Tk, D = (2, 40, 64) if axis == "batch" else (1, 70, 64)
    stride = (2 ** 31 + 8, D, D, 1) if axis == "batch" else (1, 2 ** 25 + 2 ** 24, D, 1)
    size = sum((n - 1) * s for n, s in zip((B, Tk, 1, D), stride)) + 1
    q, k, v, do = _case((B, 3, Tk, 1, 1, D), torch.bfloat16, 4)
    cache = torch.empty(size, dtype=torch.bfloat16, device="cuda")
    far = cache.as_strided((B, Tk, 1, D), stride)
    far.copy_(k.cuda())
    qd, kd, vd, dd = _cuda(q, k, v, do)
    o, l = M.cross_attention(qd, kd, vd)
    o2, l2 = M.cross_attention(qd, far, vd)
    assert torch.equal(o, o2) and torch.equal(l, l2)
    for x, y in zip(M.cross_attention_gradient(dd, qd, kd, vd, o, l), M.cross_attention_gradient(dd, qd, far, vd, o, l)):
        assert torch.equal(x, y)


def test_attention_nothing_to_attend():
    from ophelia_amd import modules as M
    for dt in DT:
        q, k, v, do = _cuda(*_case((2, 3, 0, 2, 1, 32), dt, 1))
        o, l = M.cross_attention(q, k, v)
        assert not o.any() and (l == -math.inf).all()
        dq, dk, dv = M.cross_attention_gradient(do, q, k, v, o, l)
        assert not dq.any() and dk.shape == k.shape
        q, k, v, do = _cuda(*_case((2, 0, 5, 2, 1, 32), dt, 1))
        o, l = M.cross_attention(q, k, v)
        dq, dk, dv = M.cross_attention_gradient(do, q, k, v, o, l)
        assert not dk.any() and not dv.any() and dq.shape == q.shape


def test_attention_infinite_and_nan_inputs_stay_visible():
    """A NaN that may be attended reaches the row that attends it, and no other sequence."""
    from ophelia_amd import modules as M
    q, k, v, _ = _cuda(*_case((2, 40, 60, 1, 1, 64), torch.bfloat16, 9))
    clean = M.cross_attention(q, k, v)[0]
    k[0, 17] = math.nan
    out, lse = M.cross_attention(q, k, v)
    assert out[0].isnan().all() and lse[0].isnan().all()
    assert torch.equal(out[1], clean[1])


# ---- embedding -----------------------------------------------------------------------------------------------------------------------
EMBED = [(4096, 64, 72), (4097, 300, 72), (9000, 700, 100), (40000, 40, 24), (1, 1, 1), (5, 2, 3), (33, 57, 128), (2400, 57, 128), (1000, 300, 37), (4097, 70000, 8), (5000, 3, 520), (3000, 300000, 4)]


@dtypes
@pytest.mark.parametrize("idt", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("n,V,U", EMBED, ids=str)
def test_embed(n, V, U, idt, dt):
    from ophelia_amd import modules as M
    g = torch.Generator().manual_seed(n + V)
    ids = torch.randint(-1, V + 1, (n,), generator=g).to(idt)                  # one below, one above: no row
    ids[torch.rand(n, generator=g) < 0.3] = 0
    ids[torch.rand(n, generator=g) < 0.3] = V - 1                              # a long run
    table, dout, s = _rand(1, (V, U), dt), _rand(2, (n, U), dt), math.sqrt(U)
    for pad in (True, False):
        ref, bound = O.embed(ids, table, s, pad)
        _within("lookup", M.embed_lookup(ids.cuda(), table.cuda(), scale=s, zero_pad=pad), ref, bound)
        ref, bound = O.embed_gradient(ids, dout, V, s, pad)
        _within("gradient", M.embed_gradient(ids.cuda(), dout.cuda(), V, scale=s, zero_pad=pad), ref, bound)


def test_embed_all_tokens_alike_and_none():
    from ophelia_amd import modules as M
    for n in (1, 7, 8, 9, 64, 31, 33, 5000, 8192, 8193, 20000):
        ids, dout = torch.full((n,), 7, dtype=torch.int32), _rand(3, (n, 48), torch.bfloat16)
        ref, bound = O.embed_gradient(ids, dout, 9)
        _within("gradient", M.embed_gradient(ids.cuda(), dout.cuda(), 9), ref, bound)
    none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    assert M.embed_lookup(none, torch.ones(4, 6, device="cuda")).shape == (2, 0, 6)
    assert not M.embed_gradient(none, torch.ones(2, 0, 6, device="cuda"), 4).any()
    assert not M.embed_gradient(none, torch.ones(2, 0, 6, device="cuda"), 5000).any()
    pads = torch.zeros(50, dtype=torch.int32, device="cuda")                    # only padding, whatever its gradient holds
    for V in (4, 5000):
        assert not M.embed_gradient(pads, torch.full((50, 6), math.nan, device="cuda"), V).any()


def test_embed_strides_and_far_rows():
    from ophelia_amd import modules as M
    ids = torch.tensor([[3, 1, 2], [1, 0, 4]], dtype=torch.int32, device="cuda")
    table = torch.randn(5, 2 * 24 + 1, device="cuda")[:, 25:]                    # row stride 49, odd start
    assert torch.equal(M.embed_lookup(ids, table, 0.5), M.embed_lookup(ids, table.contiguous(), 0.5))
    d = torch.randn(24, 2, 3, device="cuda").permute(1, 2, 0)                    # last axis strided
    assert torch.equal(M.embed_gradient(ids, d, 5), M.embed_gradient(ids, d.contiguous(), 5))
    far = torch.empty(4 * (2 ** 29 + 64) + 24, dtype=torch.bfloat16, device="cuda").as_strided((5, 24), (2 ** 29 + 64, 1))
    far.copy_(table)
    assert torch.equal(M.embed_lookup(ids, far), M.embed_lookup(ids, far.contiguous()))
    d16 = far[:5]
    i5 = torch.tensor([4, 4, 1, 3, 2], dtype=torch.int64, device="cuda")
    assert torch.equal(M.embed_gradient(i5, d16, 5), M.embed_gradient(i5, d16.contiguous(), 5))


# ---- gated linear recurrence ---------------------------------------------------------------------------------------------------------
@dtypes
@pytest.mark.parametrize("B,T,C", [(1, 1, 1), (2, 1, 256), (3, 7, 5), (16, 200, 256), (2, 257, 80), (1, 1030, 33), (2, 513, 129), (1, 4100, 64), (2, 9000, 20)], ids=str)
@pytest.mark.parametrize("ragged", [False, True], ids=["whole", "ragged"])
def test_recurrence(B, T, C, ragged, dt):
    from ophelia_amd import modules as M
    x, g, dh = _rand(1, (B, T, C), dt), _rand(2, (B, T, C), dt, 3.0), _rand(3, (B, T, C), dt)
    h0, dl = (None, None) if (B + T) % 2 else (_rand(4, (B, C), torch.float32), _rand(5, (B, C), torch.float32))
    lens = None
    if ragged:
        lens = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(T), dtype=torch.int32)
        lens[0] = T + 5
        if B > 1:
            lens[1] = 0
    ref, bound, ctx = O.recurrence(x, g, h0, lens)
    gref, gbound = O.recurrence_gradient(dh, dl, ctx)
    dead = ~ctx["live"].expand(B, T, C)
    for t in (x, g, dh):
        t[dead] = math.nan
    xd, gd, dd, h0d, dld, ld = _cuda(x, g, dh, h0, dl, lens)
    h, last = M.gated_recurrence(xd, gd, h0=h0d, lengths=ld)
    _within("h", h, ref[0], bound[0])
    _within("last", last, ref[1], bound[1])
    h = h.clone()
    h[dead.cuda()] = math.nan
    got = M.gated_recurrence_gradient(dd, xd, gd, h, h0=h0d, dh_last=dld, lengths=ld)
    for n, a, r, b in zip(("dx", "dgate", "dh0"), got, gref, gbound):
        _within(n, a, r, b)


def test_recurrence_gates_at_their_ends():
    """gates far out: the state is held (1 - a below every float32 step of 1) or replaced."""
    from ophelia_amd import modules as M
    x, g = _rand(1, (1, 600, 4), torch.float32), torch.tensor([-80.0, -20.0, 20.0, 80.0]).expand(1, 600, 4).contiguous()
    h0 = torch.ones(1, 4)
    ref, bound, ctx = O.recurrence(x, g, h0)
    h, last = M.gated_recurrence(x.cuda(), g.cuda(), h0=h0.cuda())
    _within("h", h, ref[0], bound[0])
    gref, gb = O.recurrence_gradient(torch.ones(1, 600, 4), None, ctx)
    for n, a, r, b in zip(("dx", "dgate", "dh0"), M.gated_recurrence_gradient(torch.ones(1, 600, 4, device="cuda"), x.cuda(), g.cuda(), h, h0=h0.cuda()), gref, gb):
        _within(n, a, r, b)


def test_recurrence_without_steps_hands_the_state_on():
    from ophelia_amd import modules as M
    for dt in DT:
        x, h0 = torch.zeros(3, 0, 5, dtype=dt, device="cuda"), torch.randn(3, 5, device="cuda")
        h, last = M.gated_recurrence(x, x, h0=h0)
        assert h.shape == (3, 0, 5) and torch.equal(last, h0)
        dx, dg, d0 = M.gated_recurrence_gradient(x, x, x, h, h0=h0, dh_last=h0)
        assert dx.shape == dg.shape == (3, 0, 5) and torch.equal(d0, h0)
        h, last = M.gated_recurrence(x[:0], x[:0])
        assert h.shape == (0, 0, 5) and last.shape == (0, 5)


def test_recurrence_steps_make_the_sequence():
    """one step at a time, the state handed on, is the whole sequence's bound; strided and time-major inputs give the same bits."""
    from ophelia_amd import modules as M
    B, T, C = 3, 40, 50
    x, g = _rand(1, (B, T, C), torch.float32), _rand(2, (B, T, C), torch.float32)
    ref, bound, _ = O.recurrence(x, g)
    xd, gd = x.cuda(), g.cuda()
    state, hs = None, []
    for t in range(T):
        h, state = M.gated_recurrence(xd[:, t:t + 1], gd[:, t:t + 1], h0=state)
        hs.append(h)
    _within("h", torch.cat(hs, 1), ref[0], bound[0])
    _within("last", state, ref[1], bound[1])
    whole = M.gated_recurrence(xd, gd)
    tm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (xd, gd)]
    both = torch.empty(B, T, 2 * C + 1, device="cuda")
    both[..., :C], both[..., C + 1:] = xd, gd
    for a, b in (tm, (both[..., :C], both[..., C + 1:])):
        h, last = M.gated_recurrence(a, b)
        assert torch.equal(h, whole[0]) and torch.equal(last, whole[1])
        d1 = M.gated_recurrence_gradient(a, a, b, h)
        for p, q in zip(d1, M.gated_recurrence_gradient(xd, xd, gd, whole[0])):
            assert torch.equal(p, q)


def test_recurrence_offsets_beyond_32_bits():
    from ophelia_amd import modules as M
    T, C, st = 70, 64, 2 ** 25 + 2 ** 24
    x, g = _cuda(_rand(1, (1, T, C), torch.bfloat16), _rand(2, (1, T, C), torch.bfloat16))
    far = torch.empty((T - 1) * st + C, dtype=torch.bfloat16, device="cuda").as_strided((1, T, C), (1, st, 1))
    far.copy_(x)
    h, last = M.gated_recurrence(x, g)
    h2, last2 = M.gated_recurrence(far, g)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    for a, b in zip(M.gated_recurrence_gradient(x, x, g, h), M.gated_recurrence_gradient(far, far, g, h)):
        assert torch.equal(a, b)


# ---- together ------------------------------------------------------------------------------------------------------------------------
def _model(M, p, ids, frames, tl, fl):
    """text -> embedding -> recurrence -> keys and values; frames -> recurrence -> queries; one attention.  Returns its result and
    what the gradient needs."""
    B, N = ids.shape
    e = M.embed_lookup(ids, p["table"], scale=4.0)
    hk, _ = M.gated_recurrence(e, p["gate"].expand_as(e), lengths=tl)
    hq, _ = M.gated_recurrence(frames, p["gate"].expand_as(frames), lengths=fl)
    q, k, v = hq.view(B, -1, 4, 16), hk.view(B, N, 4, 16)[:, :, :2], hk.view(B, N, 4, 16)[:, :, 2:]
    o, l = M.cross_attention(q, k, v, q_lens=fl, k_lens=tl)
    return e, hk, hq, q, k, v, o, l


def _model_gradient(M, p, ids, frames, tl, fl, saved, do):
    e, hk, hq, q, k, v, o, l = saved
    dq, dk, dv = M.cross_attention_gradient(do, q, k, v, o, l, q_lens=fl, k_lens=tl)
    B, N = ids.shape
    dhk = torch.cat([dk, dv], 2).view(B, N, 64)
    de, dgk, _ = M.gated_recurrence_gradient(dhk, e, p["gate"].expand_as(e), hk, lengths=tl)
    df, dgq, _ = M.gated_recurrence_gradient(dq.view_as(frames), frames, p["gate"].expand_as(frames), hq, lengths=fl)
    return M.embed_gradient(ids, de, p["table"].shape[0], scale=4.0), dgk.sum((0, 1)) + dgq.sum((0, 1)), df


def _inputs():
    g = torch.Generator().manual_seed(21)
    ids = torch.randint(1, 40, (3, 23), generator=g, dtype=torch.int32)
    tl, fl = torch.tensor([23, 9, 16], dtype=torch.int32), torch.tensor([31, 40, 12], dtype=torch.int32)
    for b in range(3):
        ids[b, tl[b]:] = 0
    p = dict(table=_rand(1, (40, 64), torch.float32, 0.3), gate=_rand(2, (64,), torch.float32))
    return p, ids, _rand(3, (3, 40, 64), torch.float32), tl, fl, _rand(4, (3, 40, 4, 16), torch.float32)


def _loss64(p, ids, frames, tl, fl, do):
    """The same model in 64 bits on the CPU: sum(out * do)."""
    table = torch.cat([torch.zeros(1, 64, dtype=O.F64), p["table"][1:]])
    e = table[ids.long()] * 4.0
    hk, hq = torch.zeros(3, 64, dtype=O.F64), torch.zeros(3, 64, dtype=O.F64)
    a = torch.sigmoid(p["gate"])
    ks, qs = [], []
    for t in range(23):
        hk = a * hk + (1 - a) * e[:, t]
        ks.append(hk)
    for t in range(40):
        hq = a * hq + (1 - a) * frames[:, t]
        qs.append(hq)
    K, Q = torch.stack(ks, 1).view(3, 23, 4, 16), torch.stack(qs, 1).view(3, 40, 4, 16)
    k, v = (x.transpose(1, 2).repeat_interleave(2, 1) for x in (K[:, :, :2], K[:, :, 2:]))
    s = Q.transpose(1, 2) @ k.transpose(2, 3) / 4.0
    s = s.masked_fill(~(torch.arange(23)[None] < tl[:, None])[:, None, None], -math.inf)
    out = (torch.softmax(s, 3) @ v).transpose(1, 2)
    return (out * do * (torch.arange(40)[None] < fl[:, None])[:, :, None, None]).sum()


def test_run_of_the_operators_and_its_gradient():
    """Result and gradient of the run, against 64 bits by the formulas (autograd) and by differences.  float32 throughout: four operators
    of at most 128 dependent roundings each are within 2^-14 of the largest element."""
    from ophelia_amd import modules as M
    p, ids, frames, tl, fl, do = _inputs()
    P = {k: t.double().requires_grad_() for k, t in p.items()}
    F = frames.double().requires_grad_()
    loss = _loss64(P, ids, F, tl, fl, do.double())
    loss.backward()
    pd = {k: t.cuda() for k, t in p.items()}
    args = (pd, ids.cuda(), frames.cuda(), tl.cuda(), fl.cuda())
    saved = _model(M, *args)
    got = _model_gradient(M, *args, saved, do.cuda())
    live = (torch.arange(40)[None] < fl[:, None])[:, :, None, None]
    assert abs((saved[6].double().cpu() * do * live).sum().item() - loss.item()) <= 2 ** -14 * (saved[6].double().cpu() * do).abs().sum().item()
    for name, g, r in zip(("table", "gate", "frames"), got, (P["table"].grad, P["gate"].grad, F.grad)):
        off = (g.double().cpu() - r).abs().max().item()
        assert off <= 2 ** -14 * r.abs().max().item(), (name, off, r.abs().max().item())
    # differences of the 64-bit loss along a random direction; the second difference bounds the step's own error
    dirs = {k: _rand(7, t.shape, torch.float64) for k, t in p.items()}
    eps = 1e-5
    at = lambda s: _loss64({k: t.double() + s * dirs[k] for k, t in p.items()}, ids, frames.double(), tl, fl, do.double()).item()
    slope = (at(eps) - at(-eps)) / (2 * eps)
    mine = sum((g.double().cpu() * dirs[k]).sum().item() for k, g in zip(("table", "gate"), got))
    size = sum((g.double().cpu() * dirs[k]).abs().sum().item() for k, g in zip(("table", "gate"), got))
    assert abs(mine - slope) <= 2 ** -14 * size + 1e-6 * abs(slope)


def test_run_is_reproducible_on_another_stream_and_in_a_graph():
    """The run twice, on a side stream, and captured: every replay has the eager call's bits for the inputs it finds, with eager work and
    synchronisation in between; two graphs of the same run replayed in turn do not disturb each other."""
    from ophelia_amd import modules as M
    p, ids, frames, tl, fl, do = _inputs()
    pd = {k: t.cuda() for k, t in p.items()}
    args, dd = (pd, ids.cuda(), frames.cuda(), tl.cuda(), fl.cuda()), do.cuda()

    def go():
        saved = _model(M, *args)
        dq, dk, dv = M.cross_attention_gradient(dd, saved[3], saved[4], saved[5], saved[6], saved[7], q_lens=args[4], k_lens=args[3])
        e = saved[0]
        de, dg, d0 = M.gated_recurrence_gradient(e, e, pd["gate"].expand_as(e), saved[1], lengths=args[3])
        return [saved[6], saved[7], dq, dk, dv, de, dg, d0, M.embed_gradient(args[1], de, 40, scale=4.0)]

    first = [t.clone() for t in go()]
    assert all(torch.equal(a, b) for a, b in zip(first, go()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = go()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, side))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = go()
        graphs.append((gr, res))
    for i in range(4):
        args[2].copy_(_rand(50 + i, frames.shape, torch.float32))
        dd.copy_(_rand(60 + i, do.shape, torch.float32))
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        want = go()
        for gr, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want)), i


def test_split_attention_in_two_graphs():
    """A call that splits the keys (it owns a workspace) in two captured graphs, replayed in turn on two streams."""
    from ophelia_amd import modules as M
    q, k, v, _ = _cuda(*_case((2, 1, 3000, 4, 1, 64), torch.bfloat16, 2))
    q2 = q.flip(3).contiguous()
    want = [M.cross_attention(x, k, v)[0].clone() for x in (q, q2)]
    graphs = []
    for x in (q, q2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = M.cross_attention(x, k, v)[0]
        graphs.append((gr, res, torch.cuda.Stream()))
    for _ in range(5):
        for gr, res, s in graphs:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for (gr, res, s), w in zip(graphs, want):
            assert torch.equal(res, w)
            res.zero_()
        torch.cuda.synchronize()


# ---- refusals that need device tensors ---------------------------------------------------------------------------------------------------
def test_refusals():
    from ophelia_amd import _lib
    from ophelia_amd import modules as M
    q, k = torch.zeros(2, 3, 4, 16, device="cuda"), torch.zeros(2, 5, 2, 16, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [lambda: M.cross_attention(q, k.half(), k), lambda: M.cross_attention(q, k, k[:, :4]), lambda: M.cross_attention(q, k.cpu(), k),
           lambda: M.cross_attention(q[0], k, k), lambda: M.cross_attention(q, k[:1], k[:1]), lambda: M.cross_attention(q, k, k, q_lens=lens.long()),
           lambda: M.cross_attention(q, k, k, k_lens=lens[:1]), lambda: M.cross_attention(q, k, k, k_lens=lens.cpu()),
           lambda: M.cross_attention(q, k, k, key_mask=torch.ones(2, 4, dtype=torch.bool, device="cuda")),
           lambda: M.cross_attention(q, k, k, key_mask=torch.ones(2, 5, device="cuda")), lambda: M.cross_attention(q.clone().requires_grad_(), k, k),
           lambda: M.cross_attention_gradient(q, q, k, k, q, torch.zeros(2, 3, 4, device="cuda")),
           lambda: M.embed_lookup(torch.zeros(3, device="cuda"), torch.zeros(4, 4, device="cuda")),
           lambda: M.embed_lookup(torch.zeros(3, dtype=torch.int32), torch.zeros(4, 4, device="cuda")),
           lambda: M.embed_lookup(lens, torch.zeros(4, device="cuda")), lambda: M.embed_gradient(lens, torch.zeros(3, 4, device="cuda"), 4),
           lambda: M.embed_gradient(lens, torch.zeros(2, 4, device="cuda"), 0),
           lambda: M.gated_recurrence(q[..., 0], k[..., 0]), lambda: M.gated_recurrence(q[0, 0], q[0, 0]),
           lambda: M.gated_recurrence(q[..., 0], q[..., 0], h0=torch.zeros(2, 4, dtype=torch.bfloat16, device="cuda")),
           lambda: M.gated_recurrence(q[..., 0], q[..., 0], lengths=lens.long())]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was not refused" % i)
    for call in (lambda: M.cross_attention(q, k[:, :, :1].expand(2, 5, 3, 16), k[:, :, :1].expand(2, 5, 3, 16)),
                 lambda: M.cross_attention(torch.zeros(1, 1, 1, 20, device="cuda"), torch.zeros(1, 1, 1, 20, device="cuda"), torch.zeros(1, 1, 1, 20, device="cuda")),
                 lambda: M.cross_attention(q, k, k, scale=-1.0), lambda: M.embed_lookup(lens, torch.zeros(4, 4, device="cuda"), scale=math.inf)):
        with pytest.raises(_lib.OpheliaHipError):
            call()


def test_synthesis_library_loaded_before_torch():
    """libophelia_hip.so loads the system's HIP runtime, torch may bring its own under another name: the operators must find torch's, also on
    a stream of torch's."""
    import subprocess
    import sys
    from conftest import ROOT
    code = ("from ophelia_amd import _lib; _lib.load(); from ophelia_amd import modules as M; "
            "import torch; s = torch.cuda.Stream(); t = torch.arange(12., device='cuda').view(4, 3); torch.cuda.synchronize();\n"
            "with torch.cuda.stream(s): r = M.embed_lookup(torch.tensor([2, 1], device='cuda'), t)\n"
            "s.synchronize(); assert r.tolist() == [[6., 7., 8.], [3., 4., 5.]], r; print('right')")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "right" in r.stdout, (r.returncode, r.stdout[-500:], r.stderr[-1500:])


def test_calls_on_two_streams_at_once():
    """Long recurrences, whose blocks wait for one another inside a launch, and split attentions and embedding gradients, queued on two streams
    without waiting: every result has the bits of the call alone."""
    from ophelia_amd import modules as M
    x = [_rand(s, (4, 6000, 192), torch.bfloat16).cuda() for s in (1, 2)]
    g = [_rand(s, (4, 6000, 192), torch.bfloat16, 2.0).cuda() for s in (3, 4)]
    q = [_rand(s, (2, 1, 8, 64), torch.bfloat16).cuda() for s in (5, 6)]
    k = [_rand(s, (2, 5000, 2, 64), torch.bfloat16).cuda() for s in (7, 8)]
    ids = [torch.randint(0, 3000, (9000,), generator=torch.Generator().manual_seed(s)).cuda() for s in (9, 10)]
    d = [_rand(s, (9000, 64), torch.bfloat16).cuda() for s in (11, 12)]

    def go(i):
        h, last = M.gated_recurrence(x[i], g[i])
        return [h, last, *M.gated_recurrence_gradient(x[i], x[i], g[i], h), *M.cross_attention(q[i], k[i], k[i]), M.embed_gradient(ids[i], d[i], 3000)]

    want = [go(i) for i in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in (0, 1)]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(go(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i])), i


@dtypes
@pytest.mark.parametrize("D", [64, 72, 128, 256])
def test_attention_padded_rows_of_split_masked_keys(D, dt):
    """A mask, and lengths that leave whole tiles of rows without a query, where the keys are split so often that the last pieces begin
    behind the keys: a padded tile reads no key and no byte of the mask."""
    from ophelia_amd import modules as M
    B, Tq, Tk = 2, 48, 2049
    q, k, v, do = _case((B, Tq, Tk, 1, 1, D), dt, 31)
    ql, kl = torch.tensor([16, 33], dtype=torch.int32), torch.tensor([Tk, 40], dtype=torch.int32)
    mask = torch.rand(B, Tk, generator=torch.Generator().manual_seed(6)) < 0.7
    out, lse, bo, bl, ctx = O.attention(q, k, v, ql, kl, mask)
    ref, bound = O.attention_gradient(do, ctx)
    qd, kd, vd, dd, qld, kld = _cuda(q, k, v, do, ql, kl)
    wide = torch.zeros(B, 2 * Tk, dtype=torch.bool, device="cuda")
    wide[:, ::2] = mask.cuda()
    for m in (mask.cuda(), wide[:, ::2]):                                  # every byte, and every other one
        o, l = M.cross_attention(qd, kd, vd, q_lens=qld, k_lens=kld, key_mask=m)
        _within("out", o, out, bo)
        _within("lse", l, lse, bl)
        for n, g, r, b in zip(("dq", "dk", "dv"), M.cross_attention_gradient(dd, qd, kd, vd, o, l, q_lens=qld, k_lens=kld, key_mask=m), ref, bound):
            _within(n, g, r, b)


@dtypes
@pytest.mark.parametrize("B,T,C", [(2, 200, 40), (2, 700, 72), (1, 3000, 24)], ids=str)
def test_recurrence_gradient_where_the_state_follows_its_input(B, T, C, dt):
    """An input that stays for a while and then moves by a step of its type: h_{t-1} - x is far smaller than h, down to less than the half step
    that h is rounded by in 16 bits, and still has to be that of the float32 state."""
    from ophelia_amd import modules as M
    step = torch.finfo(dt).eps
    gen = torch.Generator().manual_seed(T)
    moves = torch.randint(0, 3, (B, T, C), generator=gen).float() * (torch.rand(B, T, C, generator=gen) < 0.05)
    x = (1 + (moves.cumsum(1) % 64) * step).to(dt)
    g, dh, h0, dl = _rand(2, (B, T, C), dt), _rand(3, (B, T, C), dt), _rand(4, (B, C), torch.float32), _rand(5, (B, C), torch.float32)
    lens = torch.tensor([T] + [T - 61] * (B - 1), dtype=torch.int32)
    ref, bound, ctx = O.recurrence(x, g, h0, lens)
    gref, gbound = O.recurrence_gradient(dh, dl, ctx)
    xd, gd, dd, h0d, dld, ld = _cuda(x, g, dh, h0, dl, lens)
    h, last = M.gated_recurrence(xd, gd, h0=h0d, lengths=ld)
    _within("h", h, ref[0], bound[0])
    got = M.gated_recurrence_gradient(dd, xd, gd, h, h0=h0d, dh_last=dld, lengths=ld)
    for n, a, r, b in zip(("dx", "dgate", "dh0"), got, gref, gbound):
        _within(n, a, r, b)


@dtypes
@pytest.mark.parametrize("grows", [False, True], ids=["even", "growing"])
@pytest.mark.parametrize("shape", [(2, 70, 90, 2, 1, 64), (2, 200, 300, 4, 2, 128), (1, 150, 260, 2, 1, 192), (2, 5, 60, 1, 1, 32), (1, 700, 20, 2, 2, 40)], ids=str)
def test_attention_gradient_with_large_score_gradients(shape, grows, dt):
    """Score gradients beyond the range of float16 (65504) whose sums are inside it, all along and from one key and one row to the next."""
    from ophelia_amd import modules as M
    B, Tq, Tk, Hq, Hk, D = shape
    q, k, v, do = (t.float() for t in _case(shape, torch.float32, 17))
    q, k, v, do = q * 0.01, k * 0.01, v * 100, do * 7000
    if grows:
        v, do = v * torch.logspace(-3, 0, Tk)[None, :, None, None], do * torch.logspace(-3, 0, Tq)[None, :, None, None]
    q, k, v, do = (t.to(dt) for t in (q, k, v, do))
    ctx = O.attention(q, k, v)[4]
    ref, bound = O.attention_gradient(do, ctx)
    top = (ctx["P"] * (do.double().transpose(1, 2) @ ctx["V"].transpose(2, 3))).abs().max()
    assert top > 2 ** 16 and max(r.abs().max() for r in ref) < 60000, (top, [r.abs().max() for r in ref])
    qd, kd, vd, dd = _cuda(q, k, v, do)
    o, l = M.cross_attention(qd, kd, vd)
    got = M.cross_attention_gradient(dd, qd, kd, vd, o, l)
    for n, g, r, b in zip(("dq", "dk", "dv"), got, ref, bound):
        _within(n, g, r, b)


def test_refusals_of_sizes_and_scales_beyond_32_bits():
    """Expanded tensors can have any size without memory: what does not fit the library's numbers is refused as documented."""
    from ophelia_amd import _lib
    from ophelia_amd import modules as M
    ids, one = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, 1, 8, device="cuda")
    far = 2 ** 32 + 4
    for call in (lambda: M.embed_lookup(ids, one[0, 0].expand(far, 8)), lambda: M.embed_gradient(ids, one[0, 0].expand(2, 8), far),
                 lambda: M.cross_attention(one, one.expand(1, far, 1, 8), one.expand(1, far, 1, 8)),
                 lambda: M.cross_attention(one.expand(far, 1, 1, 8), one.expand(far, 1, 1, 8), one.expand(far, 1, 1, 8)),
                 lambda: M.cross_attention_gradient(one, one, one.expand(1, far, 1, 8), one.expand(1, far, 1, 8), one, one[:, :, :, 0]),
                 lambda: M.gated_recurrence(one[0].expand(1, far, 8), one[0].expand(1, far, 8)),
                 lambda: M.gated_recurrence_gradient(*[one[0].expand(1, far, 8)] * 4)):
        with pytest.raises(ValueError):
            call()
    for scale in (1e300, -1e300, 1e-60, math.inf, math.nan, 0.0):
        with pytest.raises(_lib.OpheliaHipError):
            M.cross_attention(one, one, one, scale=scale)


def test_a_refused_device_leaves_no_error_behind():
    """What the runtime answers to a device that is not there is reported by the call, and not once more by the caller's next GPU call."""
    from ophelia_amd import _lib
    lib = _lib.load_seq()
    ids, table = torch.ones(2, dtype=torch.int32, device="cuda"), torch.ones(3, 4, device="cuda")
    out = torch.zeros(2, 4, device="cuda")
    torch.cuda.synchronize()
    for device in (1000, -1):
        rc = lib.oph_seq_embed_lookup(ids.data_ptr(), 4, 2, table.data_ptr(), 4, 3, 4, 1.0, 1, 0, out.data_ptr(), device, None)
        assert rc == -3 and "device" in lib.oph_seq_last_error().decode()
        assert (table + 1).sum().item() == 24                              # torch asks for the last error after every launch
        assert not out.any()


# shapes that give a wave of every forward kernel several tiles of keys: shared tiles (with 5 or more, and a remainder), split keys, 16 rows, few rows
LONG = [(8, 130, 333, 16, 16, 64), (8, 70, 333, 32, 16, 72), (8, 130, 333, 16, 16, 128), (16, 130, 170, 8, 8, 192), (2, 33, 700, 2, 2, 64),
        (2, 40, 800, 4, 2, 128), (1, 33, 1400, 1, 1, 256), (2, 1, 900, 2, 1, 64), (2, 2, 3000, 4, 2, 128), (3, 300, 450, 1, 1, 40)]


@dtypes
@pytest.mark.parametrize("kind", ["even", "growing", "falling", "masked"])
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_attention_where_the_maximum_moves_from_tile_to_tile(shape, kind, dt):
    """Scores whose maximum rises (or falls) by more than 2^8 from one tile of keys to the next, several times along the keys, or does neither; masked: it rises,
    with whole tiles and every third key of the others left out, and ragged lengths."""
    from ophelia_amd import modules as M
    B, Tq, Tk, Hq, Hk, D = shape
    q, k, v, do = _case(shape, torch.float32, 23)
    size = torch.linspace(0.1, 20.0, Tk)[None, :, None, None]
    k = k if kind == "even" else k * (size.flip(1) if kind == "falling" else size)
    q, k, v, do = (t.to(dt) for t in (q, k, v, do))
    ql = kl = mask = None
    if kind == "masked":
        g = torch.Generator().manual_seed(3)
        ql, kl = (torch.randint(n // 2, n + 1, (B,), generator=g, dtype=torch.int32) for n in (Tq, Tk))
        mask = torch.ones(B, Tk, dtype=torch.bool)
        mask[:, ::3] = mask[:, :70] = mask[:, 128:192] = False
    out, lse, bo, bl, ctx = O.attention(q, k, v, ql, kl, mask)
    ref, bound = O.attention_gradient(do, ctx)
    qd, kd, vd, dd, qld, kld, md = _cuda(q, k, v, do, ql, kl, mask)
    o, l = M.cross_attention(qd, kd, vd, q_lens=qld, k_lens=kld, key_mask=md)
    _within("out", o, out, bo)
    _within("lse", l, lse, bl)
    for n, g, r, b in zip(("dq", "dk", "dv"), M.cross_attention_gradient(dd, qd, kd, vd, o, l, q_lens=qld, k_lens=kld, key_mask=md), ref, bound):
        _within(n, g, r, b)


@dtypes
@pytest.mark.parametrize("T", [1, 40, 600])
def test_recurrence_state_updated_in_place(T, dt):
    """The C ABI lets h0 be h_last's buffer: the state of a decoder, one block and several."""
    import ctypes as C
    from ophelia_amd import _lib
    from ophelia_amd import modules as M
    B, Ch = 3, 50
    x, g, state = _rand(1, (B, T, Ch), dt).cuda(), _rand(2, (B, T, Ch), dt).cuda(), _rand(3, (B, Ch), torch.float32).cuda()
    lens = torch.tensor([T, 0, (T + 1) // 2], dtype=torch.int32, device="cuda")
    h, last = M.gated_recurrence(x, g, h0=state, lengths=lens)
    lib, a = _lib.load_seq(), _lib.OphSeqRecur()
    out = torch.empty_like(x)
    a.x, a.gate, a.h0, a.h, a.h_last, a.lens = x.data_ptr(), g.data_ptr(), state.data_ptr(), out.data_ptr(), state.data_ptr(), lens.data_ptr()
    a.x_stride[:], a.gate_stride[:] = x.stride()[:2], g.stride()[:2]
    a.B, a.T, a.C, a.dtype = B, T, Ch, DT.index(dt)
    need = lib.oph_seq_recur_workspace(C.byref(a), 0)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    assert lib.oph_seq_recur_forward(C.byref(a), 0, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, h) and torch.equal(state, last)


@pytest.mark.parametrize("dt", DT[1:], ids=IDS[1:])
def test_long_16_bit_gradients_in_two_graphs(dt):
    """The gradients whose launches hand each other states, norms and parts through a workspace, captured twice: every replay has the eager
    call's bits for the inputs it finds, with eager work on another size in between."""
    from ophelia_amd import modules as M
    x, g, dh = (_rand(s, (2, 600, 72), dt).cuda() for s in (1, 2, 3))
    h0 = _rand(4, (2, 72), torch.float32).cuda()
    lens = torch.tensor([600, 333], dtype=torch.int32, device="cuda")
    q, k, v, do = _cuda(*_case((2, 90, 700, 4, 2, 64), dt, 5))

    def go():
        h, last = M.gated_recurrence(x, g, h0=h0, lengths=lens)
        o, l = M.cross_attention(q, k, v)
        return [h, last, *M.gated_recurrence_gradient(dh, x, g, h, h0=h0, lengths=lens), o, l, *M.cross_attention_gradient(do, q, k, v, o, l)]

    go()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = go()
        graphs.append((gr, res))
    for i in range(4):
        x.copy_(_rand(20 + i, x.shape, dt))
        do.copy_(_rand(30 + i, do.shape, dt, 10.0 ** (i + 1)))               # the last ones bring score gradients out of float16's range
        lens.copy_(torch.tensor([600 - 130 * i, 1 + 190 * i], dtype=torch.int32))
        for gr, _ in graphs:
            gr.replay()
        M.gated_recurrence_gradient(dh[:, :300], x[:, :300], g[:, :300], x[:, :300])
        torch.cuda.synchronize()
        want = go()
        for gr, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want)), i
            assert not any(r.isnan().any() for r in res)
