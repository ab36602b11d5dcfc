"""The operators' waits for copies are bounded, and what stands behind a wait
that ran out depends on its answer: read from the kernels' sources, as no test
makes a copy fail."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "stream-mm2026_b200" / "csrc"
CALL = re.compile(r"\b(?:bar_wait|warp_wait)\s*\(")


def _statements(name):
    """The statements of a source, without comments, that call a wait."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", (CSRC / name).read_text(), flags=re.S)
    return [" ".join(s.split()) for s in re.split(r"[;{}]", text) if CALL.search(s)]


def _answer_is_dropped(statement):
    # the end of a `for (...;...;...)` ahead of it
    depth = 0
    for i, c in enumerate(statement):
        depth += (c == "(") - (c == ")")
        if depth < 0:
            return _answer_is_dropped(statement[i + 1:].strip())
    # `if (...) wait(...)` drops it as well as `wait(...)` alone does
    head = re.sub(r"^(?:(?:else|do)\b|(?:if|for|while)\s*\((?:[^()]|\([^()]*\))*\))+", "", statement).strip()
    return CALL.match(head) is not None


def test_dropped_answers_are_found():
    for text in ("bar_wait(&b, 0)", "else bar_wait(&b, 0)", "if (x) warp_wait(&b[f(k)], 1)",
                 "++k) bar_wait(&b[k % n], 0)"):
        assert _answer_is_dropped(text)
    for text in ("(void)bar_wait(&b, 0)", "if (!bar_wait(&b, 0)) lost = true", "ok &= bar_wait(&b, 0)",
                 "return __all_sync(m, bar_wait(b, p))", "else if (!lost && warp_wait(&b, 0)) next()"):
        assert not _answer_is_dropped(text)


@pytest.mark.parametrize("name", ["mdq_distill.cu", "mdq_norm.cuh"])
def test_every_wait_is_answered(name):
    found = [s for s in _statements(name) if "__forceinline__" not in s]
    assert found
    assert not [s for s in found if _answer_is_dropped(s)]


def test_waits_end():
    """One loop with a limit holds every wait of the operators on a barrier of copies."""
    text = (CSRC / "mdq_ops.cuh").read_text()
    assert re.search(r"\[\[nodiscard\]\][^;{]*bar_wait", text)
    assert text.count("mbarrier.try_wait") == 1 and "for (int i = 0; i < 1 << 22; ++i)" in text
    for path in CSRC.glob("mdq_*"):
        if path.name.startswith(("mdq_distill", "mdq_norm", "mdq_embed")):
            assert "try_wait" not in path.read_text() and "test_wait" not in path.read_text()
