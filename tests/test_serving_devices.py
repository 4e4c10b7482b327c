"""The serving operators and the device that is current, on a stand-in for the CUDA runtime with two devices
(tests/fake_cuda.c, preloaded in a process of its own): every launch, attribute and occupancy question of a call goes to its
context's device, and the caller's device is current again afterwards, also where the call is refused."""
import json
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

WORKER = r"""
import ctypes as C, json
from agxforge_b200 import _native as N
L = N.lib()
fake = C.CDLL(None)
fake.fake_log.restype = C.c_char_p
def current():
    d = C.c_int()
    fake.cudaGetDevice(C.byref(d))
    return d.value
ctx = []
for d in (0, 1):
    p = C.c_void_p()
    assert L.agxc_init(d, C.byref(p)) == 0, L.agxc_last_error()
    ctx.append(p)
P = 1 << 20                                              # an address that nothing reads
def cache(hd=128, kvh=8, pages=4096, page=64):
    return N.Kv4Cache(P, pages, kvh, hd, page)
def append(hd=128):
    W = 32 * hd
    return N.Kv4AppendArgs(cache(hd), P, W, N.F32, 5, 16, P, P, P, P, 64, None, None, None, 1e-6, 1.0, P, N.F16)
def attention(B, n, H, mp, hd=128, ws=1 << 40):
    return N.Kv4AttentionArgs(cache(hd), P, P, N.F16, B, n, H, P, mp, mp, P, P, ws)
def sample(dtype=N.F32):
    return N.SampleArgs(P, 50257, dtype, 7, 50257, P, 1.0, 0.9, 0.0, 50, None, None, None, None, P, P)
calls = {}
for hd in (64, 128):
    calls["append %d" % hd] = lambda c, s, hd=hd: L.agxc_kv4_append_dev(c, C.byref(append(hd)), s)
    calls["rows %d" % hd] = lambda c, s, hd=hd: L.agxc_kv4_rows_dev(c, C.byref(cache(hd)), P, 9, P, P, s)
    for name, shape in [("few", (1, 1, 16, 28)), ("line", (64, 1, 32, 128)), ("chunk", (2, 256, 32, 36))]:
        calls["%s %d" % (name, hd)] = lambda c, s, a=shape, hd=hd: L.agxc_kv4_attention_dev(c, C.byref(attention(*a, hd)), s)
        calls["workspace %s %d" % (name, hd)] = \
            lambda c, s, a=shape, hd=hd: min(0, L.agxc_kv4_attention_workspace(c, C.byref(attention(*a, hd))))
    calls["refused %d" % hd] = lambda c, s, hd=hd: L.agxc_kv4_attention_dev(c, C.byref(attention(64, 1, 32, 128, hd, 8)), s)
for t in (N.F32, N.F16, N.BF16):
    calls["sample %d" % t] = lambda c, s, t=t: L.agxc_sample_dev(c, C.byref(sample(t)), s)
out = []
for name, call in calls.items():
    for here, there in ((0, 1), (1, 0), (0, 0), (1, 1)):
        for stream in (None, 1):
            fake.cudaSetDevice(here)
            fake.fake_clear()
            rc = call(ctx[there], stream)
            out.append(dict(name=name, here=here, there=there, stream=stream, rc=rc, after=current(), sets=fake.fake_sets(),
                            log=[l.split() for l in fake.fake_log().decode().splitlines()]))
lost = []
for name, call in calls.items():                          # a device that cannot be made current
    fake.cudaSetDevice(0)
    fake.fake_clear()
    fake.fake_fail_set(1)
    rc = call(ctx[1], None)
    fake.fake_fail_set(0)
    lost.append(dict(name=name, rc=rc, after=current(), log=fake.fake_log().decode()))
print("RESULT " + json.dumps([out, lost]))
"""


@pytest.fixture(scope="module")
def result(tmp_path_factory):
    from agxforge_b200 import build
    build.build()
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    so = str(tmp_path_factory.mktemp("fake") / "fake_cuda.so")
    subprocess.run([cc, "-shared", "-fPIC", "-O1", "-o", so, os.path.join(ROOT, "tests", "fake_cuda.c")], check=True)
    p = subprocess.run([sys.executable, "-c", WORKER], cwd=ROOT, capture_output=True, text=True,
                       env=dict(os.environ, LD_PRELOAD=so, PYTHONPATH=ROOT))
    assert p.returncode == 0, p.stderr[-3000:]
    return json.loads(p.stdout.split("RESULT ")[1])


def test_calls_go_to_their_contexts_device(result):
    for r in result[0]:
        where = (r["name"], r["here"], r["there"], r["stream"])
        assert r["rc"] == (-1 if "refused" in r["name"] else 0), where
        assert all(int(line[1]) == r["there"] for line in r["log"]), (where, r["log"])
        launches = [line for line in r["log"] if line[0] == "launch"]
        want = 0 if "workspace" in r["name"] or "refused" in r["name"] else 2 if "line" in r["name"] else 1
        assert len(launches) == want, (where, r["log"])
        # no stream: the context's own
        assert all(int(line[3]) == (1 if r["stream"] else 0x5000 + r["there"]) for line in launches), where


def test_the_callers_device_is_current_again(result):
    for r in result[0]:
        assert r["after"] == r["here"], r["name"]
        assert r["sets"] == (0 if r["here"] == r["there"] else 2), r["name"]


def test_a_device_that_cannot_be_made_current(result):
    for r in result[1]:
        assert r["rc"] < 0 and r["after"] == 0 and r["log"] == "", r["name"]


def test_paged_model_makes_its_device_current(monkeypatch):
    """The model's own steps go through calls that take the current device's stream."""
    import contextlib

    import torch

    from agxforge.inference import paged
    from agxforge.kernels import kv4
    stack = [0]

    @contextlib.contextmanager
    def device(d):
        stack.append(d)
        yield
        stack.pop()

    seen = []

    class Shape:
        VOCAB, EPS = 100, 1e-6

    def rows(ids, n):
        seen.append(("rows", stack[-1]))
        for s in ids:
            m.seqs[s]["held"] += n
        return torch.zeros(len(ids), 4)

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda d=None: None)
    monkeypatch.setattr(kv4, "check_errors", lambda device=0: seen.append(("check", stack[-1])))
    monkeypatch.setattr(paged.sampling, "sample", lambda lg, u, *a: (
        seen.append(("sample", stack[-1])), (torch.full((lg.shape[0],), 3), torch.ones(lg.shape[0])))[1])
    m = paged.PagedModel.__new__(paged.PagedModel)
    m.device, m.shape, m.seqs, m._next, m.spare, m.page_size = 5, Shape, {}, 0, [], 16
    m.head = m.final_gain = None
    monkeypatch.setattr(m, "_rows", rows, raising=False)
    monkeypatch.setattr(m, "_gemv", lambda *a, **k: (seen.append(("gemv", stack[-1])), torch.zeros(a[1].shape[0], 100))[1],
                        raising=False)
    s = m.add([1, 2, 3])
    m.logits()
    m.seqs[s]["tokens"].append(7)
    assert m.step([0.5]) == {s: (3, 1.0)}
    assert {"rows", "gemv", "sample"} <= {what for what, _ in seen}
    assert all(d == 5 for _, d in seen), seen
    assert stack == [0]
