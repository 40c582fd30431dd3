"""Inline assembly that copies to or from memory says so, or the compiler may move plain accesses of the same bytes across it."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "memory_b200", "csrc")
WRITES = r"\b(cp\.async\.(ca|cg|bulk)(?!\.prefetch)|st\.(shared|global)|red\.|atom\.|mbarrier\.(arrive|try_wait|test_wait)|barrier\.cluster)"


def _statements(text):
    """The text of every asm statement: from `asm` to its closing parenthesis."""
    for m in re.finditer(r"\basm\b\s*(volatile)?\s*\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.start():i]


def test_the_scan_sees_a_missing_clobber():
    bad = 'asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(f(x)), "l"(y));'
    found = list(_statements("int a; " + bad + " int b;"))
    assert found == [bad[:-1]] and re.search(WRITES, found[0]) and '"memory"' not in found[0]


def test_asynchronous_copies_and_barriers_clobber_memory():
    seen, bad = 0, []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        for s in _statements(open(path).read()):
            if re.search(WRITES, s):
                seen += 1
                if '"memory"' not in s or "volatile" not in s:
                    bad.append((os.path.basename(path), s))
    assert seen > 10 and not bad, bad
