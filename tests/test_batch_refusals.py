"""What the batch operators (qp_batch_rope_append, qp_batch_attn, qp_verify_drafts) refuse, checked without a GPU: the C entry points
validate before anything is launched, the Python face before it looks for a stream.  Pointers here are never followed."""
import ctypes

import pytest
import torch

from quickvideo_amd import native

A = 1 << 20                      # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    return native.load_library()


@pytest.fixture(scope="module")
def ctx():
    class Ctx(ctypes.Structure):  # struct qp_ctx {device, cus, lds_per_cu, lt}
        _fields_ = [("device", ctypes.c_int), ("cus", ctypes.c_int), ("lds", ctypes.c_int), ("lt", ctypes.c_void_p)]
    c = Ctx(0, 256, 65536, None)
    return ctypes.addressof(c), c


APPEND = dict(qkv=A, cos=A, sin=A, batch=2, t_max=3, seq_len=A, n_new=None, n_q=28, n_kv=4, head_dim=128, q_out=A + (1 << 24), k_pages=A, v_pages=A,
              page_stride=4 * 16 * 128, n_pages=9, page_size=16, table=A, max_pages=4)
ATTN = dict(q=A, k_prefix=A, v_prefix=A, stride=200 * 128, prefix_len=200, k_pages=A, v_pages=A, page_stride=4 * 16 * 128, n_pages=9, page_size=16, table=A,
            max_pages=4, seq_len=A, n_new=None, batch=2, t_max=3, n_q=28, n_kv=4, head_dim=128, scale=0.1, out=A, ws=A, ws_bytes=1 << 30)
VERIFY = dict(logits=A, f32=1, seq_stride=5000, row_stride=1000, drafts=A, n_draft=None, probs=None, pss=0, prs=0, u=A, batch=2, t_max=4, vocab=1000,
              temperature=1.0, accepted=A, tokens=A, ws=A, ws_bytes=1 << 24)


def call(fn, ctx, base, **change):
    args = dict(base)
    args.update(change)
    return fn(ctx[0], *args.values(), None)


@pytest.mark.parametrize("change,status,word", [
    (dict(qkv=None), -1, "NULL"), (dict(seq_len=None), -1, "NULL"), (dict(table=None), -1, "NULL"), (dict(q_out=None), -1, "NULL"),
    (dict(head_dim=64), -2, "head_dim"), (dict(batch=0), -1, "batch"), (dict(t_max=0), -1, "t_max"), (dict(batch=1 << 9, t_max=1 << 9), -2, "65536"),
    (dict(n_q=30), -1, "multiple"), (dict(n_kv=0), -1, "multiple"), (dict(n_q=2048, n_kv=1), -2, "1024"), (dict(n_pages=0), -1, "n_pages"),
    (dict(page_size=0), -1, "page_size"), (dict(max_pages=0), -1, "max_pages"), (dict(page_size=1 << 16, max_pages=1 << 16, page_stride=1 << 40), -2, "2^30"),
    (dict(page_stride=4 * 16 * 128 - 8), -1, "page_stride"), (dict(page_stride=4 * 16 * 128 + 4), -1, "page_stride"), (dict(k_pages=A + 8), -1, "aligned"),
    (dict(qkv=A + 2), -1, "alignment"), (dict(cos=A + 4), -1, "alignment"), (dict(q_out=A + 4096), -1, "overlaps"),
])
def test_append_refuses(lib, ctx, change, status, word):
    assert call(lib.qp_batch_rope_append, ctx, APPEND, **change) == status
    assert word in lib.qp_last_error().decode()


def test_no_context(lib):
    for fn, base in ((lib.qp_batch_rope_append, APPEND), (lib.qp_batch_attn, ATTN), (lib.qp_verify_drafts, VERIFY)):
        assert fn(None, *base.values(), None) == -1 and "NULL" in lib.qp_last_error().decode()


@pytest.mark.parametrize("change,status,word", [
    (dict(q=None), -1, "NULL"), (dict(ws=None), -1, "NULL"), (dict(k_prefix=None), -1, "without prefix"), (dict(v_prefix=None), -1, "without prefix"),
    (dict(head_dim=80), -2, "head_dim"), (dict(prefix_len=-1), -1, "prefix_len"), (dict(stride=199 * 128), -1, "prefix_head_stride"),
    (dict(stride=200 * 128 + 4), -1, "prefix_head_stride"), (dict(prefix_len=(1 << 30) + 1, stride=1 << 40), -2, "2^30"), (dict(scale=0.0), -1, "scale"),
    (dict(scale=-1.0), -1, "scale"), (dict(scale=float("nan")), -1, "scale"), (dict(scale=float("inf")), -1, "scale"), (dict(out=A + 8), -1, "alignment"),
    (dict(k_prefix=A + 2), -1, "alignment"), (dict(ws_bytes=1000), -4, "workspace"), (dict(batch=70000, t_max=1), -2, "65536"), (dict(n_q=27), -1, "multiple"),
    (dict(page_size=17), -1, "page_stride"),
])
def test_attn_refuses(lib, ctx, change, status, word):
    assert call(lib.qp_batch_attn, ctx, ATTN, **change) == status
    assert word in lib.qp_last_error().decode()


@pytest.mark.parametrize("change,status,word", [
    (dict(logits=None), -1, "NULL"), (dict(accepted=None), -1, "NULL"), (dict(tokens=None), -1, "NULL"), (dict(drafts=None), -1, "drafts"),
    (dict(u=None), -1, "random"), (dict(batch=0), -1, "batch"), (dict(batch=65536), -1, "batch"), (dict(t_max=-1), -2, "t_max"), (dict(t_max=256), -2, "t_max"),
    (dict(vocab=0), -2, "vocab"), (dict(vocab=4194305, row_stride=1 << 30, seq_stride=1 << 30), -2, "vocab"), (dict(temperature=-0.5), -1, "temperature"),
    (dict(temperature=float("nan")), -1, "temperature"), (dict(temperature=float("inf")), -1, "temperature"), (dict(row_stride=999), -1, "strides"),
    (dict(seq_stride=999), -1, "strides"), (dict(probs=A, pss=4000, prs=999), -1, "draft_probs"), (dict(probs=A, pss=999, prs=1000), -1, "draft_probs"),
    (dict(logits=A + 2), -1, "alignment"), (dict(logits=A + 1, f32=0), -1, "alignment"), (dict(probs=A + 2, pss=4000, prs=1000), -1, "alignment"),
    (dict(ws=A + 4), -1, "alignment"), (dict(ws_bytes=100), -4, "workspace"),
])
def test_verify_refuses(lib, ctx, change, status, word):
    assert call(lib.qp_verify_drafts, ctx, VERIFY, **change) == status
    assert word in lib.qp_last_error().decode()


def test_workspace_sizes(lib, ctx):
    good = lib.qp_batch_attn_workspace_bytes(ctx[0], 4, 1, 11535, 256, 28, 4)
    assert good > 0
    for bad in ((0, 1, 10, 16, 28, 4), (4, 0, 10, 16, 28, 4), (4, 1, -1, 16, 28, 4), (4, 1, 10, 0, 28, 4), (4, 1, 10, 16, 27, 4), (70000, 1, 10, 16, 28, 4)):
        assert lib.qp_batch_attn_workspace_bytes(ctx[0], *bad) == 0
    assert lib.qp_batch_attn_workspace_bytes(None, 4, 1, 10, 16, 28, 4) == 0
    assert lib.qp_verify_drafts_workspace_bytes(3, 4, 152064) > lib.qp_verify_drafts_workspace_bytes(3, 0, 1) > 0
    for bad in ((0, 4, 10), (1, -1, 10), (1, 256, 10), (1, 4, 0), (65536, 0, 10), (1, 0, 4194305)):
        assert lib.qp_verify_drafts_workspace_bytes(*bad) == 0


@pytest.fixture
def ops(ctx):
    o = object.__new__(native.QuickPrefillOps)          # no GPU: everything below is refused before a pointer is taken
    o.lib, o.ctx, o.device = native.load_library(), ctypes.c_void_p(None), torch.device("cuda", 0)
    o._bind_face()
    o._dev, o._stream_of = -1, lambda dev: 0            # -1: where torch says CPU tensors are
    yield o
    o.ctx = None


def batch_tensors(B=2, T=3, hq=4, hkv=2, ps=4, pages=6, width=3):
    bf = torch.bfloat16
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)                                                           # noqa: E731
    return dict(qkv=torch.zeros(B, T, (hq + 2 * hkv) * 128, dtype=bf), cos=torch.zeros(B, T, 64, dtype=bf), sin=torch.zeros(B, T, 64, dtype=bf), seq_len=i32(B),
                n_new=i32(B), table=i32(B, width), k_pages=torch.zeros(pages, hkv, ps, 128, dtype=bf), v_pages=torch.zeros(pages, hkv, ps, 128, dtype=bf),
                n_q=hq, n_kv=hkv, head_dim=128, q_out=torch.zeros(B, T, hq, 128, dtype=bf))


@pytest.mark.parametrize("name,make,word", [
    ("qkv", lambda t: t.float(), "float32"), ("qkv", lambda t: t[:, :, :-1], "shape"), ("cos", lambda t: t[:, :2], "shape"), ("sin", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), "contiguous"), ("q_out", lambda t: t[:, :, :3], "shape"),
    ("seq_len", lambda t: t.long(), "int64"), ("n_new", lambda t: t[:1], "shape"), ("table", lambda t: t.float(), "float32"), ("table", lambda t: t.t(), "shape"),
    ("k_pages", lambda t: t.half(), "float16"), ("v_pages", lambda t: t[:, :, :2], "shape"), ("v_pages", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), "page"),
    ("v_pages", lambda t: torch.cat([t, t], 1)[:, :2], "page"), ("qkv", lambda t: t, "is on cpu"),
])
def test_python_append_refuses(ops, name, make, word):
    kw = batch_tensors()
    kw[name] = make(kw[name])
    if word == "is on cpu":
        ops._dev = 0
    with pytest.raises(ValueError, match=word):
        ops.batch_rope_append(*kw.values())


@pytest.mark.parametrize("name,make,word", [
    ("logits", lambda t: t.double(), "float64"), ("logits", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), "rows must be contiguous"),
    ("drafts", lambda t: t.int(), "int32"), ("drafts", lambda t: t[:, :1], "shape"), ("probs", lambda t: t.double(), "float64"), ("probs", lambda t: t[:, :, :5], "shape"),
    ("u", lambda t: t[:, :1], "shape"), ("accepted", lambda t: t.long(), "int64"), ("tokens", lambda t: t[:, :2].contiguous(), "shape"), ("logits", lambda t: t, "is on cpu"),
])
def test_python_verify_refuses(ops, name, make, word):
    B, T, V = 2, 2, 7
    kw = dict(logits=torch.zeros(B, T + 1, V), drafts=torch.zeros(B, T, dtype=torch.int64), n_draft=None, probs=torch.zeros(B, T, V), u=torch.zeros(B, T + 1),
              temperature=1.0, accepted=torch.zeros(B, dtype=torch.int32), tokens=torch.zeros(B, T + 1, dtype=torch.int64), ws=torch.zeros(4096, dtype=torch.uint8))
    kw[name] = make(kw[name])
    if word == "is on cpu":
        ops._dev = 0
    with pytest.raises(ValueError, match=word):
        ops.verify_drafts(*kw.values())


def test_python_workspaces_refuse(ops, ctx):
    ops.ctx = ctypes.c_void_p(ctx[0])
    with pytest.raises(ValueError, match="no batch"):
        ops.batch_attn_workspace(0, 1, 10, 16, 28, 4)
    with pytest.raises(ValueError, match="no verification"):
        ops.verify_drafts_workspace(1, 256, 1000)


def test_python_good_calls_reach_the_library(ops):
    """Well-formed tensors pass the face and end at the library's own first check (no context here)."""
    with pytest.raises(ValueError, match="qp_batch_rope_append: NULL"):
        ops.batch_rope_append(*batch_tensors().values())
    kw = batch_tensors()
    q, kp = torch.zeros(2, 3, 4, 128, dtype=torch.bfloat16), torch.zeros(2, 10, 128, dtype=torch.bfloat16)
    attn = [q, kp, kp, 1280, 10, kw["k_pages"], kw["v_pages"], kw["table"], kw["seq_len"], None, 4, 2, 128, 0.1, q.clone(), torch.zeros(64, dtype=torch.uint8)]
    with pytest.raises(ValueError, match="qp_batch_attn: NULL"):
        ops.batch_attn(*attn)
    for at, bad, word in ((4, 11, "fewer"), (3, 1408, "fewer"), (1, kp.float(), "float32"), (0, q[:, :2], "contiguous"), (14, q.transpose(0, 1), "shape"), (15, torch.zeros(8, 8).t(), "contiguous"),
                          (5, kw["k_pages"][0], "n_pages"), (10, 8, "shape")):
        with pytest.raises(ValueError, match=word):
            ops.batch_attn(*[bad if i == at else v for i, v in enumerate(attn)])
    with pytest.raises(ValueError, match="qp_verify_drafts: NULL"):
        ops.verify_drafts(torch.zeros(2, 3, 7), torch.zeros(2, 2, dtype=torch.int64), None, None, torch.zeros(2, 3), 1.0, torch.zeros(2, dtype=torch.int32),
                          torch.zeros(2, 3, dtype=torch.int64), torch.zeros(4096, dtype=torch.uint8))
    with pytest.raises(TypeError):
        ops._face.batch_attn(1, 2)
    for name in ("qkv", "table", "n_new"):
        kw = batch_tensors()
        kw[name] = "no tensor"
        with pytest.raises((ValueError, AttributeError)):
            ops.batch_rope_append(*kw.values())


def test_missing_face_fails_loudly(monkeypatch):
    import sys
    monkeypatch.setitem(sys.modules, "quickvideo_amd._qp_torch", None)
    monkeypatch.delattr("quickvideo_amd._qp_torch", raising=False)
    with pytest.raises(native.QuickPrefillUnavailable, match="_qp_torch"):
        native.load_face()


def test_tensors_without_plain_memory_are_refused(ops):
    """A sparse tensor's is_contiguous() throws in C++: it must come back as a Python error, not end the process."""
    kw = batch_tensors()
    B, T, hq, hkv = 2, 3, 4, 2
    q, kp = torch.zeros(B, T, hq, 128, dtype=torch.bfloat16), torch.zeros(hkv, 10, 128, dtype=torch.bfloat16)
    sparse = torch.zeros(8, 8).to_sparse()
    attn = [q, kp, kp, 1280, 10, kw["k_pages"], kw["v_pages"], kw["table"], kw["seq_len"], kw["n_new"], hq, hkv, 128, 0.1, q.clone(), torch.zeros(1 << 16, dtype=torch.uint8)]
    for at in (0, 1, 5, 7, 15):
        bad = sparse if at == 15 else attn[at].to_sparse()
        with pytest.raises((ValueError, RuntimeError)):
            ops.batch_attn(*[bad if i == at else v for i, v in enumerate(attn)])
    with pytest.raises((ValueError, RuntimeError)):
        ops.verify_drafts(torch.zeros(2, 3, 7), torch.zeros(2, 2, dtype=torch.int64), None, None, torch.zeros(2, 3), 1.0, torch.zeros(2, dtype=torch.int32),
                          torch.zeros(2, 3, dtype=torch.int64), sparse)
    with pytest.raises((ValueError, RuntimeError)):
        ops.batch_rope_append(*(kw | {"qkv": kw["qkv"].to_sparse()}).values())


@pytest.mark.parametrize("batch,t_max,n_q,n_kv,prefix,fits", [
    (65536, 1, 1024, 1024, 200, False), (32768, 2, 1024, 1024, 200, False), (65536, 1, 128, 128, 200, True), (65536, 1, 128, 128, 1000, False),
    (65536, 1, 64, 64, 200, True), (65536, 1, 64, 64, 1000, True), (65536, 1, 28, 4, 200, True), (16, 4096, 64, 8, 200, True), (1, 65536, 64, 64, 1000, True),
])
def test_batches_that_no_launch_takes_are_refused(lib, ctx, batch, t_max, n_q, n_kv, prefix, fits):
    """grid x threads of a launch stay below 2^32: larger batches are refused before the first launch, and the workspace query says so.  65536 one-token
    sequences x 128 key heads are 2^23 workgroups of the pages: of 256 threads over a short prefix, of 512 over a longer one."""
    need = lib.qp_batch_attn_workspace_bytes(ctx[0], batch, t_max, prefix, 64, n_q, n_kv)
    assert (need > 0) == fits
    change = dict(batch=batch, t_max=t_max, n_q=n_q, n_kv=n_kv, prefix_len=prefix, stride=prefix * 128, page_stride=n_kv * 16 * 128)
    if fits:
        assert call(lib.qp_batch_attn, ctx, ATTN, **change, ws_bytes=need - 1) == -4
    else:
        assert call(lib.qp_batch_attn, ctx, ATTN, **change, ws_bytes=1 << 60) == -2
        assert "2^32" in lib.qp_last_error().decode()


@pytest.mark.parametrize("scale,good", [(1e8, True), (1.01e8, False), (1e9, False), (3e38, False), (1e-30, True)])
def test_scales_that_leave_an_empty_range_finite(lib, ctx, scale, good):
    """The running maximum of a row that has seen nothing is -1e30; a scale that makes -1e30 * scale * log2(e) infinite turned such a range into NaN."""
    assert call(lib.qp_batch_attn, ctx, ATTN, scale=scale, ws_bytes=1000) == (-4 if good else -1)
    assert ("workspace" if good else "scale") in lib.qp_last_error().decode()


@pytest.mark.parametrize("shift,good", [(0, True), (16, False), (-16, False), (2 * 3 * 28 * 256 - 16, False), (2 * 3 * 28 * 256, True), (-2 * 3 * 28 * 256, True)])
def test_out_is_q_or_apart_from_it(lib, ctx, shift, good):
    assert call(lib.qp_batch_attn, ctx, ATTN, out=A + shift, ws_bytes=1000) == (-4 if good else -1)
    assert ("workspace" if good else "overlaps") in lib.qp_last_error().decode()


def test_the_other_operators_need_no_face(monkeypatch):
    """An operator object comes up and works with the library alone; only a call of the batch operators asks for the module, and says how to build it."""
    import sys

    class Lib:
        """the library's entry points that construction calls, without a device"""
        def __getattr__(self, name):
            return {"qp_create": lambda out, device: 0, "qp_select_workspace_bytes": lambda n: 16, "qp_destroy": lambda ctx: None,
                    "qp_decode_advance": lambda *a: 0}[name]

    monkeypatch.setitem(sys.modules, "quickvideo_amd._qp_torch", None)
    monkeypatch.delattr("quickvideo_amd._qp_torch", raising=False)
    monkeypatch.setattr(native, "load_library", lambda *a, **k: Lib())
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(native.QuickPrefillOps, "_stream", staticmethod(lambda: 0))
    ops = native.QuickPrefillOps(torch.device("cpu"))
    ops.decode_advance(torch.zeros(2, dtype=torch.int64))
    with pytest.raises(native.QuickPrefillUnavailable, match="make -C quickvideo_amd/csrc face"):
        ops.batch_rope_append(*batch_tensors().values())


def test_the_library_builds_without_torch():
    """`make` asks neither g++ nor Python for anything (programs in C build the library alone); `make face` builds the module."""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.abspath(native.__file__)), "csrc")
    plan = lambda *goal: subprocess.run(["make", "-Bn", "-C", csrc, "PYTHON=echo no-python", *goal], capture_output=True, text=True, check=True).stdout   # noqa: E731
    assert "libquickprefill.so" in plan() and "g++" not in plan() and "no-python" not in plan() and "_qp_torch" not in plan()
    assert "g++" in plan("face") and "_qp_torch.so" in plan("face")
