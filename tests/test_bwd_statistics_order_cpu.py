"""The items of the attention's backward pass start beside the kernel that computes the row statistics: nothing that runs
before their wait for it may touch these.  Read from the source, because on a GPU a read that comes too early mostly finds
what an earlier call of the same inputs left."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mod-dit_b200", "csrc", "sparse_attn_bwd.cu")
WAIT = "griddepcontrol.wait"
STATISTICS = re.compile(r"\b(nlse|ndelta)\b")


def plain(text):
    return re.sub(r"//[^\n]*", "", text)


def braces(text, start):
    """The text from `start` through the block that opens behind it."""
    depth, i = 0, text.index("{", start)
    for j in range(i, len(text)):
        depth += {"{": 1, "}": -1}.get(text[j], 0)
        if depth == 0:
            return text[start:j + 1]
    raise AssertionError("unbalanced")


def functions(text):
    """name -> bodies of the device functions and of the methods (several structs have one of a name)."""
    found = {}
    for m in re.finditer(r"__device__ (?:__forceinline__|__noinline__) [\w:<> ]+?\b(\w+)\(", text):
        found.setdefault(m.group(1), []).append(braces(text, m.start()))
    return found


def test_statistics_are_read_behind_the_wait():
    text = plain(open(SOURCE).read())
    assert text.count(WAIT) == 1
    at = text.index("sparse_attn_bwd_kernel(")
    before, behind = braces(text, text.index(") {", at)).split(WAIT)
    bodies = functions(text)
    assert {"item_of", "expand", "visible", "load", "produce", "compute", "issue"} <= set(bodies)

    def reached(body, seen):
        for name in re.findall(r"\b(\w+)\s*(?:<[\w, ]+>)?\(", body):
            if name in bodies and name not in seen:
                seen.add(name)
                for b in bodies[name]:
                    reached(b, seen)
        return seen

    early = reached(before, set())
    assert {"item_of", "expand", "visible", "load"} <= early and not {"produce", "compute", "issue"} & early
    assert not STATISTICS.search(before)
    for name in early:
        for body in bodies[name]:
            assert not STATISTICS.search(body), name
    assert any(STATISTICS.search(b) for name in reached(behind, set()) for b in bodies[name])
