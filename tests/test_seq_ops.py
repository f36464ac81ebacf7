"""libophelia_seq.so without a GPU: it exports what include/ophelia_seq.h declares, refuses bad arguments before it looks for a device, and
fails loudly where there is none."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT


@pytest.fixture(scope="module")
def lib():
    from ophelia_amd import _lib
    if not os.path.exists(_lib.SEQ_LIBPATH):
        _lib.build()
    return _lib.load_seq()


def test_library_exports_every_declared_symbol(lib):
    from ophelia_amd import _lib
    txt = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ophelia_seq.h")).read(), flags=re.S)
    syms = set(re.findall(r"\b(oph_seq_[a-z0-9_]+)\s*\(", txt))
    assert syms == set(_lib.SEQ_SIGNATURES)
    assert lib.oph_seq_abi_version() == 1


def _attn(**over):
    from ophelia_amd import _lib
    a = _lib.OphSeqAttn()
    for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"):
        setattr(a, n, 4096)                      # never followed: every call below is refused
    a.B, a.Tq, a.Tk, a.Hq, a.Hk, a.D, a.dtype, a.scale = 2, 3, 5, 4, 2, 64, 1, 0.125
    for n, x in over.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("over,word", [(dict(dtype=3), "dtype"), (dict(B=-1), "negative"), (dict(Tk=-1), "negative"), (dict(Hq=3), "multiple"),
                                       (dict(Hk=0), "multiple"), (dict(D=12), "head size"), (dict(D=264), "head size"), (dict(D=0), "head size"),
                                       (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
                                       (dict(scale=float("inf")), "scale"), (dict(Tq=2 ** 31 - 1), "too many"), (dict(q=None), "NULL"),
                                       (dict(k=None), "NULL"), (dict(out=None), "NULL"), (dict(Tk=100000, Tq=1), "workspace"),
                                       (dict(Tk=100000, Tq=1, workspace=4096, workspace_bytes=64), "workspace"),
                                       (dict(Tk=100000, Tq=1, workspace=4100, workspace_bytes=1 << 40), "workspace")], ids=str)
def test_attention_refusals(lib, over, word):
    a = _attn(**over)
    for call in (lib.oph_seq_attn_forward, lib.oph_seq_attn_gradient):
        rc = call(C.byref(a), 0, None)
        assert rc in (-1, -4) and word in lib.oph_seq_last_error().decode(), (rc, lib.oph_seq_last_error())
    if word in ("dtype", "negative", "multiple", "head size", "scale", "too many"):
        assert lib.oph_seq_attn_workspace(C.byref(a), 0) < 0


def test_empty_calls_and_null_arguments(lib):
    assert lib.oph_seq_attn_forward(None, 0, None) == -1 and lib.oph_seq_recur_forward(None, 0, None) == -1
    a = _attn(B=0)
    assert lib.oph_seq_attn_forward(C.byref(a), 0, None) == 0 and lib.oph_seq_attn_gradient(C.byref(a), 0, None) == 0
    assert lib.oph_seq_embed_lookup(None, 4, 0, None, 8, 5, 8, 1.0, 1, 0, None, 0, None) == 0


@pytest.mark.parametrize("args,word", [((4096, 2, 5, 4096, 8, 5, 8, 1.0, 1, 0), "bytes"), ((4096, 4, -1, 4096, 8, 5, 8, 1.0, 1, 0), "ids"),
                                       ((4096, 4, 5, 4096, 8, 0, 8, 1.0, 1, 0), "table"), ((4096, 4, 5, 4096, 8, 5, 0, 1.0, 1, 0), "table"),
                                       ((4096, 4, 5, 4096, -8, 5, 8, 1.0, 1, 0), "stride"), ((4096, 4, 5, 4096, 8, 5, 8, float("nan"), 1, 0), "scale"),
                                       ((4096, 4, 5, 4096, 8, 5, 8, 1.0, 1, 9), "dtype"), ((None, 4, 5, 4096, 8, 5, 8, 1.0, 1, 0), "NULL"),
                                       ((4096, 4, 5, None, 8, 5, 8, 1.0, 1, 0), "NULL")], ids=str)
def test_embedding_refusals(lib, args, word):
    assert lib.oph_seq_embed_lookup(*args, 4096, 0, None) == -1 and word in lib.oph_seq_last_error().decode()
    assert lib.oph_seq_embed_gradient(*args, 4096, 4096, 1 << 40, 0, None) == -1 and word in lib.oph_seq_last_error().decode()


def test_embedding_workspace_is_checked(lib):
    ok = (4096, 4, 500, 4096, 8, 5000, 8, 1.0, 1, 0, 4096)
    need = lib.oph_seq_embed_workspace(500, 5000, 8)
    assert need > 0
    for ws, size in ((None, need), (4096, need - 1), (4104, need)):
        assert lib.oph_seq_embed_gradient(*ok, ws, size, 0, None) == -1 and "workspace" in lib.oph_seq_last_error().decode()


@pytest.mark.parametrize("over,word", [(dict(dtype=-1), "dtype"), (dict(B=-1), "size"), (dict(T=-1), "size"), (dict(C=0), "size"), (dict(x=None), "NULL"),
                                       (dict(gate=None), "NULL"), (dict(h=None), "NULL"), (dict(T=2 ** 31 - 1), "too large")], ids=str)
def test_recurrence_refusals(lib, over, word):
    from ophelia_amd import _lib
    a = _lib.OphSeqRecur()
    for n in ("x", "gate", "h", "h_last", "dh", "dx", "dgate"):
        setattr(a, n, 4096)
    a.B, a.T, a.C, a.dtype = 2, 3, 4, 0
    for n, v in over.items():
        setattr(a, n, v)
    for call in (lib.oph_seq_recur_forward, lib.oph_seq_recur_gradient):
        assert call(C.byref(a), 0, None) in (-1, -4) and word in lib.oph_seq_last_error().decode()


def test_no_cpu_fallback():
    from ophelia_amd import modules as M
    q = torch.zeros(1, 2, 1, 8)
    for call in (lambda: M.cross_attention(q, q, q), lambda: M.embed_lookup(torch.zeros(3, dtype=torch.int32), torch.zeros(4, 4)),
                 lambda: M.embed_gradient(torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4), 4),
                 lambda: M.gated_recurrence(torch.zeros(1, 2, 3), torch.zeros(1, 2, 3)),
                 lambda: M.cross_attention_gradient(q, q, q, q, q, torch.zeros(1, 1, 2)),
                 lambda: M.gated_recurrence_gradient(*[torch.zeros(1, 2, 3)] * 4)):
        with pytest.raises(ValueError, match="GPU only"):
            call()
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        M.cross_attention(q.double(), q.double(), q.double())


def test_without_a_device_the_library_says_so(lib):
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    a = _attn()
    assert lib.oph_seq_attn_forward(C.byref(a), 0, None) == -3 and "HIP device" in lib.oph_seq_last_error().decode()


def test_product_sources_of_the_operators_stand_alone():
    """no oracle, and packed float32 instructions switched off for this library (some of their forms have given wrong results)"""
    src = open(os.path.join(ROOT, "ophelia_amd", "device_ops.py")).read()
    assert "oracle" not in src
    assert "-packed-fp32-ops" in open(os.path.join(ROOT, "ophelia_amd", "_lib.py")).read()


def test_packed_arguments_match_the_structures():
    from ophelia_amd import _lib, device_ops
    assert device_ops._ATTN.size == C.sizeof(_lib.OphSeqAttn) and device_ops._RECUR.size == C.sizeof(_lib.OphSeqRecur)
    a = _lib.OphSeqAttn.from_buffer_copy(device_ops._ATTN.pack(*range(12), *range(100, 114), 200, 201, *range(300, 307), 0.5))
    assert (a.q or 0, a.mask, list(a.q_stride), list(a.dout_stride), list(a.mask_stride)) == (0, 11, [100, 101, 102], [109, 110, 111], [112, 113])
    assert (a.workspace, a.workspace_bytes, a.B, a.Hk, a.dtype, a.scale) == (200, 201, 300, 304, 306, 0.5)
    r = _lib.OphSeqRecur.from_buffer_copy(device_ops._RECUR.pack(*range(11), *range(100, 108), 200, 201, *range(300, 304)))
    assert (r.gate, r.lens, list(r.dh_stride), r.workspace, r.workspace_bytes, r.B, r.dtype) == (1, 10, [106, 107], 200, 201, 300, 303)


def test_split_spans_stay_inside_their_axis(tmp_path):
    """The spans of a split axis and the places their flags are read from (csrc/oph_split.h), compiled for the CPU: in order, whole, inside the
    axis, also where the rounded-up pieces of a padded tile begin behind it and where the last one's end passes 32 bits."""
    src = tmp_path / "spans.cpp"
    src.write_text(r'''
#include "oph_split.h"
#include <cstdio>
#include <initializer_list>
using namespace ophseq;
static long bad = 0, seen = 0;
static void look(int n, int tile, int nsplit) {
    int at = 0;
    for (int s = 0; s < nsplit; ++s)
        for (int live = 0; live < 2; ++live) {
            const Span x = split_span(n, tile, nsplit, s, live);
            bad += x.beg < 0 || x.beg > x.end || x.end > n || (!live && x.end != x.beg);
            if (live) { bad += x.beg != at || (x.beg < n && x.beg % tile); at = x.end; }
            for (int wave = 0; wave < 8; ++wave)                     // a wave's first tile, there or not
                for (int lane = 0; lane < 64; lane += 21) {
                    const int i = flag_index(x.beg + wave * tile, lane, x.end), want = x.beg + wave * tile + lane;
                    ++seen;
                    bad += i >= n || i < -1 || (want < x.end && i != want) || (x.beg + wave * tile >= x.end && i != -1);
                }
        }
    bad += at != n;
}
int main() {
    const int tiles[] = {8, 16, 32, 64}, few[] = {0, 1, 7, 16, 17, 150, 2049, 8197, 32772};
    for (int tile : tiles) {
        for (int n = 0; n < 700; n += 1 + n / 40)
            for (int ns = 1; ns <= 256; ns += 1 + ns / 8) look(n, tile, ns);
        for (int n : few)
            for (int ns = 1; ns <= 256; ++ns) look(n, tile, ns);
        for (int n : {2147482743, 2147482000, 2147480000})
            for (int ns : {1, 3, 16, 255, 256}) look(n, tile, ns);
    }
    std::printf("%ld looked at, %ld bad\n", seen, bad);
    return bad != 0;
}
''')
    exe = str(tmp_path / "spans")
    # signed overflow ends the program: a sum that leaves 32 bits is found even where the result happens to look right
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-I", os.path.join(ROOT, "ophelia_amd", "csrc"),
                    str(src), "-o", exe], check=True, timeout=120)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.stdout[-500:], r.stderr[-1500:])


def test_sizes_beyond_32_bits_are_refused():
    """The C ABI takes sizes as 32-bit numbers: 2^32 + 4 rows must not arrive as 4."""
    from ophelia_amd import device_ops
    from ophelia_amd import modules as M
    ids, dout = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4)
    for vocab in (2 ** 32 + 4, 2 ** 31, 0, -1):
        with pytest.raises(ValueError, match="vocab"):
            M.embed_gradient(ids, dout, vocab)
    assert device_ops._sizes("x", (3, 2 ** 31 - 1)) == (3, 2 ** 31 - 1)
    with pytest.raises(ValueError, match="2147483648"):
        device_ops._sizes("x", (3, 2 ** 31))


def test_forward_mode_tangents_are_refused():
    """A dual tensor does not require a gradient: its tangent must not get lost in silence, under no_grad() neither."""
    from ophelia_amd import device_ops
    device_ops._torch or device_ops._setup()
    ad = torch.autograd.forward_ad
    look = lambda t: device_ops._like(torch, "q", t, torch.float32, t.device, t.shape)
    with ad.dual_level():
        plain, dual = torch.ones(2, 3), ad.make_dual(torch.ones(2, 3), torch.ones(2, 3))
        assert look(plain) is plain and look(ad.unpack_dual(dual).primal).shape == (2, 3)
        with pytest.raises(ValueError, match="tangent"):
            look(dual)
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
            look(dual)
    with pytest.raises(ValueError, match="gradient"):
        look(torch.ones(2, requires_grad=True))
    with torch.no_grad():
        assert look(torch.ones(2, requires_grad=True)).shape == (2,)


@pytest.mark.parametrize("over", [dict(B=2, Hq=1, Hk=1, D=8, Tq=1200000000, Tk=1), dict(B=9000, Hq=1000, Hk=1000, Tq=1, Tk=1),
                                  dict(B=2, Hq=1, Hk=1, D=8, Tq=1, Tk=1200000000), dict(B=1, Hq=1, Hk=1, D=136, dtype=0, Tq=300000000, Tk=1),
                                  dict(B=2, Hq=1, Hk=1, D=136, Tq=1, Tk=600000000)], ids=str)
def test_attention_refuses_what_one_launch_does_not_hold(lib, over):
    """A launch has less than 2^32 threads: what needs more is refused before anything is launched, not half way through a gradient.  Long
    keys do not bound the forward, nor long rows of fp32 heads above 128."""
    a = _attn(workspace=4096, workspace_bytes=1 << 50, **over)
    assert lib.oph_seq_attn_gradient(C.byref(a), 0, None) == -4 and "too many" in lib.oph_seq_last_error().decode()
    assert lib.oph_seq_attn_workspace(C.byref(a), 1) == -4
    if over["Tq"] == 1 and over["Tk"] > 1 or over.get("dtype") == 0:
        assert lib.oph_seq_attn_workspace(C.byref(a), 0) >= 0
    else:
        assert lib.oph_seq_attn_forward(C.byref(a), 0, None) == -4


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_recurrence_workspace_is_checked(lib, dtype):
    """One block needs none; longer sequences do, and in 16 bits the gradient more than the forward."""
    from ophelia_amd import _lib
    a = _lib.OphSeqRecur()
    for n in ("x", "gate", "h", "h_last", "dh", "dx", "dgate"):
        setattr(a, n, 4096)
    a.B, a.T, a.C, a.dtype = 2, 256, 40, dtype
    assert lib.oph_seq_recur_workspace(C.byref(a), 0) == lib.oph_seq_recur_workspace(C.byref(a), 1) == 0
    a.T = 257
    need = [lib.oph_seq_recur_workspace(C.byref(a), g) for g in (0, 1)]
    assert need[0] > 0 and (need[1] == need[0] if dtype == 0 else need[1] > 2 * need[0])
    for g, call in enumerate((lib.oph_seq_recur_forward, lib.oph_seq_recur_gradient)):
        for ws, size in ((None, need[g]), (4096, need[g] - 1), (4104, need[g])):
            a.workspace, a.workspace_bytes = ws, size
            assert call(C.byref(a), 0, None) == -1 and "workspace" in lib.oph_seq_last_error().decode()
