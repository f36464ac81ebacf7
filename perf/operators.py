"""The device operators of a text-to-frames model as measurable cases: embedding lookup and gradient, gated linear recurrence and
gradient, cross attention (whole sequences, single frames) and gradient -- each in its plain form (elementary torch operations in
fp32, rounded once at the end) and through ophelia_amd.modules (`own`)."""
import math
import random

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one decoder frame of 16 utterances against 150 encoder states of one 256-wide head (lj_tutorial sizes): latency
        dict(name="frame_fp32", op="attention", dtype="float32", B=16, Tq=1, Tk=150, Hq=1, Hk=1, D=256, ragged=True, masked=False),
        # one token of 8 sequences against long encoder states, heads in groups of four: one pass over the states
        dict(name="token_long_bf16", op="attention", dtype="bfloat16", B=8, Tq=1, Tk=16384, Hq=32, Hk=8, D=128, ragged=True, masked=False),
        # teacher-forced frames over their text (lj_tutorial sizes, ragged batch): training's and validation's forward
        dict(name="frames_fp32", op="attention", dtype="float32", B=16, Tq=200, Tk=150, Hq=1, Hk=1, D=256, ragged=True, masked=False),
        # long sequences of both sides, grouped heads: matrix-rate bound
        dict(name="long_bf16", op="attention", dtype="bfloat16", B=4, Tq=4096, Tk=4096, Hq=16, Hk=4, D=128, ragged=False, masked=False),
        # gradient at the training sizes of frames_fp32
        dict(name="frames_grad_fp32", op="attention_gradient", dtype="float32", B=16, Tq=200, Tk=150, Hq=1, Hk=1, D=256, ragged=True,
             masked=False),
        # gradient of a long decoder over a short, masked text; odd lengths
        dict(name="short_text_grad_fp16", op="attention_gradient", dtype="float16", B=6, Tq=2999, Tk=333, Hq=8, Hk=4, D=64, ragged=True,
             masked=True),
        # gradient of long sequences of both sides
        dict(name="long_grad_bf16", op="attention_gradient", dtype="bfloat16", B=2, Tq=4096, Tk=4096, Hq=16, Hk=4, D=128, ragged=False,
             masked=False),
        # a batch of long texts through a sub-word table
        dict(name="lookup_bf16", op="embed", dtype="bfloat16", n=32768, vocab=32000, units=1024, zipf=True),
        # the gradient of a phone table (16 texts of 150 letters, 57 rows of 128): every row is hit often
        dict(name="phones_grad_fp32", op="embed_gradient", dtype="float32", n=2400, vocab=57, units=128, zipf=False),
        # the gradient of a sub-word table: frequent tokens thousands of times, most rows never
        dict(name="words_grad_bf16", op="embed_gradient", dtype="bfloat16", n=32768, vocab=32000, units=1024, zipf=True),
        # recurrence over the mel frames of a training batch (lj_tutorial sizes)
        dict(name="recurrence_fp32", op="recurrence", dtype="float32", B=16, T=200, C=256, ragged=True),
        # a training pass of the recurrence, forward and gradient, over long sequences
        dict(name="recurrence_train_bf16", op="recurrence_train", dtype="bfloat16", B=4, T=16384, C=1024, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    op = rng.choice(["attention", "attention", "attention_gradient", "attention_gradient", "embed", "embed_gradient", "recurrence",
                     "recurrence_train"])
    if op.startswith("attention"):
        while True:
            token = op == "attention" and rng.random() < 0.4
            Hk = rng.choice([1, 1, 2, 3, 4, 8])
            c = dict(op=op, dtype=dtype, B=_log(rng, 1, 16), Tq=rng.choice([1, 1, 2, 5]) if token else _log(rng, 8, 4096),
                     Tk=_log(rng, 1, 32768 if token else 4096), Hq=Hk * rng.choice([1, 1, 2, 3, 4, 8]), Hk=Hk,
                     D=rng.choice([16, 32, 40, 64, 80, 128, 128, 192, 256]), ragged=rng.random() < 0.6, masked=rng.random() < 0.3)
            products = c["B"] * c["Tq"] * c["Tk"] * c["Hq"] * c["D"] * (4 if dtype == "float32" else 1)
            products *= 2.5 if op != "attention" else 1
            if products <= 4 * 4096 * 4096 * 16 * 128 and c["B"] * c["Tk"] * c["Hk"] * c["D"] <= 8 * 16384 * 8 * 128:
                return c
    if op.startswith("embed"):
        while True:
            c = dict(op=op, dtype=dtype, n=_log(rng, 1, 65536), vocab=_log(rng, 2, 65536), units=8 * _log(rng, 1, 256),
                     zipf=rng.random() < 0.5)
            if (c["n"] + c["vocab"]) * c["units"] <= 65536 * 1024:
                return c
    while True:
        c = dict(op=op, dtype=dtype, B=_log(rng, 1, 32), T=_log(rng, 1, 32768), C=rng.choice([1, 8, 8, 8]) * _log(rng, 1, 256),
                 ragged=rng.random() < 0.5)
        if c["B"] * c["T"] * c["C"] <= 4 * 16384 * 1024:
            return c


def _lengths(case, of, n):
    """Ragged lengths as a sorted-by-nothing batch has them: between a third of the longest and all of it, one at the full length."""
    if not case["ragged"]:
        return None
    r = random.Random("%s %d %d" % (of, n, case["B"]))
    full = r.randrange(case["B"])
    return [n if b == full else r.randint((n + 2) // 3, n) for b in range(case["B"])]


def _device(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = _TYPES[case["dtype"]]
    op = case["op"]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    s = {"case": case}
    if op.startswith("attention"):
        B, Tq, Tk, Hq, Hk, D = (case[k] for k in ("B", "Tq", "Tk", "Hq", "Hk", "D"))
        s["q"], s["k"], s["v"] = randn(B, Tq, Hq, D), randn(B, Tk, Hk, D), randn(B, Tk, Hk, D)
        s["q_lens"] = _device(_lengths(case, "q", Tq))
        s["k_lens"] = _device(_lengths(case, "k", Tk))
        s["key_mask"] = torch.rand(B, Tk, generator=g, device="cuda") < 0.9 if case["masked"] else None
        if op == "attention_gradient":
            s["dout"] = randn(B, Tq, Hq, D)
            s["out"], s["lse"] = _attention(s)
    elif op.startswith("embed"):
        n, V, U = case["n"], case["vocab"], case["units"]
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        rank = torch.exp(u * math.log(V)).long() - 1 if case["zipf"] else (u * V).long()      # log-uniform ranks: Zipf's law
        s["ids"] = rank.clamp(0, V - 1).int()
        s["scale"] = math.sqrt(U)
        if op == "embed":
            s["table"] = randn(V, U, scale=U ** -0.5)
        else:
            s["dout"] = randn(n, U)
    else:
        B, T, C = case["B"], case["T"], case["C"]
        s["x"], s["gate"] = randn(B, T, C), randn(B, T, C, scale=2.0)
        s["h0"] = torch.randn(B, C, generator=g, device="cuda")
        s["lens"] = _device(_lengths(case, "t", T))
        if op == "recurrence_train":
            s["dh"] = randn(B, T, C)
            s["dh_last"] = torch.randn(B, C, generator=g, device="cuda")
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _valid(lens, B, n):
    at = torch.arange(n, device="cuda")
    return torch.ones(B, n, dtype=torch.bool, device="cuda") if lens is None else at[None, :] < lens[:, None]


def _heads(x, G=1):
    """(B, T, H, D) -> (B, H * G, T, D) in fp32, contiguous."""
    x = x.float().transpose(1, 2)
    return x.repeat_interleave(G, dim=1).contiguous() if G > 1 else x.contiguous()


def _scores(s):
    """fp32 scores with -inf where nothing may be attended, and the validity of queries and keys."""
    case = s["case"]
    B, Tq, Tk, G = case["B"], case["Tq"], case["Tk"], case["Hq"] // case["Hk"]
    keys = _valid(s["k_lens"], B, Tk)
    if s["key_mask"] is not None:
        keys = keys & s["key_mask"]
    rows = _valid(s["q_lens"], B, Tq)
    kt = s["k"].float().permute(0, 2, 3, 1).repeat_interleave(G, dim=1).contiguous()
    S = torch.matmul(_heads(s["q"]), kt) * (case["D"] ** -0.5)
    S.masked_fill_(~keys[:, None, None, :], -math.inf)
    S.masked_fill_(~rows[:, None, :, None], -math.inf)
    return S, rows, keys


def _attention(s):
    case = s["case"]
    S, rows, keys = _scores(s)
    m = S.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    P = torch.exp(S - m)
    l = P.sum(-1, keepdim=True)
    v = torch.where(keys[:, :, None, None], s["v"].float(), 0.0)
    o = torch.matmul(P, _heads(v, case["Hq"] // case["Hk"])) / torch.where(l > 0, l, 1.0)
    lse = torch.where(l > 0, m + torch.log(l), -math.inf)[..., 0]
    return o.transpose(1, 2).contiguous().to(s["q"].dtype), lse


def _attention_gradient(s):
    case = s["case"]
    B, Tk, Hk, D, t = case["B"], case["Tk"], case["Hk"], case["D"], s["q"].dtype
    G = case["Hq"] // Hk
    S, rows, keys = _scores(s)
    lse = s["lse"][..., None]
    P = torch.where(torch.isinf(lse), 0.0, torch.exp(S - lse))
    del S
    do = _heads(torch.where(rows[:, :, None, None], s["dout"].float(), 0.0))
    delta = (do * _heads(s["out"])).sum(-1, keepdim=True)
    v = torch.where(keys[:, :, None, None], s["v"].float(), 0.0)
    vt = v.permute(0, 2, 3, 1).repeat_interleave(G, dim=1).contiguous()
    dv = torch.matmul(P.transpose(2, 3).contiguous(), do)
    dS = (torch.matmul(do, vt) - delta) * P * (D ** -0.5)
    del P
    k = torch.where(keys[:, :, None, None], s["k"].float(), 0.0)
    q = _heads(torch.where(rows[:, :, None, None], s["q"].float(), 0.0))
    dq = torch.matmul(dS, _heads(k, G)).transpose(1, 2).contiguous()
    dk = torch.matmul(dS.transpose(2, 3).contiguous(), q)

    def group(x):
        return x.view(B, Hk, G, Tk, D).sum(2).transpose(1, 2).contiguous().to(t)

    return dq.to(t), group(dk), group(dv)


def _embed(s):
    rows = s["table"].float()[s["ids"].long()] * s["scale"]
    return torch.where((s["ids"] == 0)[:, None], 0.0, rows).to(s["table"].dtype)


def _embed_gradient(s):
    V, dout = s["case"]["vocab"], s["dout"]
    rows = torch.where((s["ids"] == 0)[:, None], 0.0, dout.float() * s["scale"])
    return torch.zeros(V, dout.shape[1], device="cuda").index_add_(0, s["ids"].long(), rows).to(dout.dtype)


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t over dim 1 by doubling: after step k every element holds its window of 2^k steps."""
    step, T = 1, a.shape[1]
    while step < T:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _gates(s):
    """Gate and input in fp32; behind a sequence's end the gate is 1 and the input 0, so that the state stays."""
    B, T = s["case"]["B"], s["case"]["T"]
    live = _valid(s["lens"], B, T)[:, :, None]
    return torch.where(live, torch.sigmoid(s["gate"].float()), 1.0), torch.where(live, s["x"].float(), 0.0), live


def _recurrence(s):
    a, x, live = _gates(s)
    b = (1 - a) * x
    b[:, 0] += a[:, 0] * s["h0"]
    h = _scan(a, b)
    return torch.where(live, h, 0.0).to(s["x"].dtype), h[:, -1].clone(), h


def _recurrence_train(s):
    h, last, full = _recurrence(s)
    a, x, live = _gates(s)
    dh = torch.where(live, s["dh"].float(), 0.0)
    dh[:, -1] += s["dh_last"]
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)          # the gate of the step that follows
    l = _scan(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([s["h0"][:, None], full[:, :-1]], 1)
    dx = torch.where(live, (1 - a) * l, 0.0)
    dgate = torch.where(live, a * (1 - a) * (before - x) * l, 0.0)
    return h, last, dx.to(h.dtype), dgate.to(h.dtype), a[:, 0] * l[:, 0]


def _plain(s):
    op = s["case"]["op"]
    if op == "attention":
        return _attention(s)
    if op == "attention_gradient":
        return _attention_gradient(s)
    if op == "embed":
        return _embed(s)
    if op == "embed_gradient":
        return _embed_gradient(s)
    if op == "recurrence":
        return _recurrence(s)[:2]
    return _recurrence_train(s)


# ---- the framework's operators ----------------------------------------------------------------------------------------------
def run(state):
    if not own:
        return _plain(state)
    from ophelia_amd import modules as M
    s, op = state, state["case"]["op"]
    if op == "attention":
        return M.cross_attention(s["q"], s["k"], s["v"], q_lens=s["q_lens"], k_lens=s["k_lens"], key_mask=s["key_mask"])
    if op == "attention_gradient":
        return M.cross_attention_gradient(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], q_lens=s["q_lens"],
                                          k_lens=s["k_lens"], key_mask=s["key_mask"])
    if op == "embed":
        return M.embed_lookup(s["ids"], s["table"], scale=s["scale"])
    if op == "embed_gradient":
        return M.embed_gradient(s["ids"], s["dout"], s["case"]["vocab"], scale=s["scale"])
    h, last = M.gated_recurrence(s["x"], s["gate"], h0=s["h0"], lengths=s["lens"])
    if op == "recurrence":
        return h, last
    return (h, last) + tuple(M.gated_recurrence_gradient(s["dh"], s["x"], s["gate"], h, h0=s["h0"], dh_last=s["dh_last"],
                                                         lengths=s["lens"]))


def work(case):
    op = case["op"]
    e = 4 if case["dtype"] == "float32" else 2
    if op.startswith("attention"):
        B, Tq, Tk, Hq, Hk, D = (case[k] for k in ("B", "Tq", "Tk", "Hq", "Hk", "D"))
        ql = _lengths(case, "q", Tq) or [Tq] * B
        kl = _lengths(case, "k", Tk) or [Tk] * B
        pairs = Hq * sum(a * b for a, b in zip(ql, kl)) * D
        rows, keys = sum(ql) * Hq * D * e, sum(kl) * Hk * D * e
        if op == "attention":                            # q, k, v in; out whole, lse
            return {"bytes": rows + 2 * keys + B * Tq * Hq * (D * e + 4), "flops": 4 * pairs}
        return {"bytes": 3 * rows + 2 * keys + sum(ql) * Hq * 4 + B * Tq * Hq * D * e + 2 * B * Tk * Hk * D * e, "flops": 10 * pairs}
    if op == "embed":
        n, U = case["n"], case["units"]                  # rows that several ids share are read once
        return {"bytes": n * 4 + min(n, case["vocab"]) * U * e + n * U * e, "flops": n * U}
    if op == "embed_gradient":
        n, U = case["n"], case["units"]
        return {"bytes": n * 4 + n * U * e + case["vocab"] * U * e, "flops": 2 * n * U}
    B, T, C = case["B"], case["T"], case["C"]
    steps = sum(_lengths(case, "t", T) or [T] * B) * C
    forward = 2 * steps * e + B * T * C * e + 2 * B * C * 4
    if op == "recurrence":
        return {"bytes": forward, "flops": 8 * steps}
    return {"bytes": forward + 4 * steps * e + 2 * B * T * C * e + 3 * B * C * 4, "flops": 24 * steps}


# ---- the operators' definitions in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op.startswith("attention"):
        B, Tq, Tk, Hq, Hk, D = (case[k] for k in ("B", "Tq", "Tk", "Hq", "Hk", "D"))
        if B * Tq * Tk * Hq * D > 2 * 10 ** 11:
            return None
        G, scale = Hq // Hk, 1.0 / math.sqrt(D)
        out = torch.zeros(B, Tq, Hq, D, dtype=f64, device="cuda")
        lse = torch.full((B, Hq, Tq), -math.inf, dtype=f64, device="cuda")
        dq, dk, dv = torch.zeros_like(out), *(torch.zeros(B, Tk, Hk, D, dtype=f64, device="cuda") for _ in range(2))
        ql, kl = _lengths(case, "q", Tq) or [Tq] * B, _lengths(case, "k", Tk) or [Tk] * B
        for b in range(B):
            idx = torch.arange(kl[b], device="cuda")
            if s["key_mask"] is not None:
                idx = idx[s["key_mask"][b, :kl[b]]]
            if idx.numel() == 0:
                continue
            n = ql[b]
            for h in range(Hq):
                q, k, v = s["q"][b, :n, h].to(f64), s["k"][b, idx, h // G].to(f64), s["v"][b, idx, h // G].to(f64)
                z = q @ k.T.contiguous() * scale
                lz = torch.logsumexp(z, 1)
                p = torch.exp(z - lz[:, None])
                out[b, :n, h], lse[b, h, :n] = p @ v, lz
                if op == "attention_gradient":
                    do = s["dout"][b, :n, h].to(f64)
                    dp = do @ v.T.contiguous()
                    dz = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                    dq[b, :n, h] = dz @ k
                    dk[b, idx, h // G] += dz.T.contiguous() @ q
                    dv[b, idx, h // G] += p.T.contiguous() @ do
        return (out, lse) if op == "attention" else (dq, dk, dv)
    if op == "embed":
        table = s["table"].to(f64).clone()
        table[0] = 0
        return torch.index_select(table, 0, s["ids"].long()) * s["scale"]
    if op == "embed_gradient":
        # sums of consecutive rows in token order, as differences of running sums would lose digits: one segment after the other
        order = torch.argsort(s["ids"].long(), stable=True)
        counts = torch.bincount(s["ids"].long(), minlength=case["vocab"])
        rows = s["dout"].to(f64)[order]
        grad = torch.segment_reduce(rows, "sum", lengths=counts, unsafe=True, initial=0.0) * s["scale"]
        grad[0] = 0
        return grad
    B, T, C = case["B"], case["T"], case["C"]
    lens = torch.tensor(_lengths(case, "t", T) or [T] * B, device="cuda")[:, None]
    x, z = s["x"].to(f64), s["gate"].to(f64)
    a = 1 / (1 + torch.exp(-z))
    keep = 1 / (1 + torch.exp(z))
    h = torch.zeros(B, T + 1, C, dtype=f64, device="cuda")
    h[:, 0] = s["h0"].to(f64)
    for t in range(T):
        h[:, t + 1] = torch.where(t < lens, a[:, t] * h[:, t] + keep[:, t] * x[:, t], h[:, t])
    live = (torch.arange(T, device="cuda")[None, :] < lens)[:, :, None]
    last = h[:, T].clone()
    states = torch.where(live, h[:, 1:], 0.0)
    if op == "recurrence":
        return states, last
    l = s["dh_last"].to(f64)
    dx, dgate = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T - 1, -1, -1):
        now = t < lens
        g = l + s["dh"][:, t].to(f64)
        dx[:, t] = torch.where(now, keep[:, t] * g, 0.0)
        dgate[:, t] = torch.where(now, a[:, t] * keep[:, t] * (h[:, t] - x[:, t]) * g, 0.0)
        l = torch.where(now, a[:, t] * g, l)
    return states, last, dx, dgate, l
