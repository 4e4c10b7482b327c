"""The bounded waits of the serving kernels, by reading their sources: a wait whose lanes answer for themselves may give up
on some lanes of a warp only, and the next warp-wide operation then waits for the others. So every wait is one of the warp's
(mbar_wait_warp, mbar_wait_quiet_warp) or stands inside a vote (ok_all), and no answer is dropped but those of the waits for
copies and MMAs on the way out."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "agxforge_b200", "csrc")
# waits on the way out, after which nothing reads what they waited for
LAST = [r"mbar_wait_quiet_warp\(&full\[x % S\]", r"mbar_wait_quiet_warp\(&br\.raw_full\[x % kRaw\]",
        r"mbar_wait_quiet_warp\(&br\.drained", r"mbar_wait_warp\(&sh\.copied\[c\]"]


def _source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def _inside(text, at, opener):
    """Is position `at` between the parentheses of a call of `opener`?"""
    for m in re.finditer(re.escape(opener) + r"\(", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        if m.start() < at < i:
            return True
    return False


@pytest.mark.parametrize("name", ["kv4_attention.cu", "kv4_chunk.cu", "sampling.cu"])
def test_every_wait_is_the_warps(name):
    text = _source(name)
    waits = list(re.finditer(r"\bmbar_wait_(bounded|quiet)\(", text))
    assert all(_inside(text, m.start(), "ok_all") for m in waits), [text[m.start():m.start() + 60] for m in waits]
    assert waits or "mbar_wait_warp(" in text


@pytest.mark.parametrize("name", ["kv4_attention.cu", "kv4_chunk.cu", "sampling.cu"])
def test_no_answer_is_dropped(name):
    text = _source(name)
    for m in re.finditer(r"\bmbar_wait_\w+\(", text):
        before = text[:m.start()].rstrip()
        if before[-1] in ";{})":                       # a statement of its own
            assert any(re.match(p, text[m.start():]) for p in LAST), text[m.start():m.start() + 60]


def test_a_warps_wait_votes():
    """Both leave on a vote alone, whether the phase completed or the limit passed."""
    text = _source("common.cuh")
    for name in ("mbar_wait_warp", "mbar_wait_quiet_warp"):
        body = text[text.index("bool %s(" % name):]
        body = body[:body.index("__device__", 1)]
        for m in re.finditer(r"\bmbar_try_wait\w*\(", body):
            assert _inside(body, m.start(), "__all_sync")
        ways = re.findall(r"if \((.*)\) (?:return true;|\{)", body)
        assert len(ways) == 3 and all("__all_sync" in w or "__any_sync" in w for w in ways)


def test_a_row_that_did_not_come_gives_no_token():
    """Sampling: a copy that did not land in time makes the row's token -1, after a second wait for it."""
    text = _source("sampling.cu")
    assert "came = came && mbar_wait_warp(" in text and "__syncthreads_or(!came)" in text
    lost = text[text.index("if (!whole) {"):]
    lost = lost[:lost.index("return;")]
    assert "mbar_wait_warp(&sh.copied[c]" in lost and "p.token[b] = -1;" in lost


@pytest.mark.parametrize("name", ["kv4_attention.cu", "kv4_chunk.cu", "sampling.cu"])
def test_what_launches_remember_is_atomic(name):
    """Calls of different threads meet in the tables of what a device takes (the binding lets go of the interpreter's lock)."""
    kept = re.findall(r"\bstatic (?!constexpr|const |_)([\w:<> ]+?) (\w+)\[", _source(name))
    assert kept and all(kind.startswith("std::atomic<") for kind, _ in kept), kept
