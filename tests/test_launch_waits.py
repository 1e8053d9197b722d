"""Kernels whose launches overlap the one before them wait for it (``grid_wait`` in ``csrc/ptx.cuh``) before they read global memory.  What is
read as constant, by ``__ldg`` or through ``const __restrict__`` parameters, may be read early by a compiler, but not through a
pointer that comes out of the wait: read here from the sources, since a wrong order need not show in results."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).parent.parent / "piper_b200" / "csrc"
SOURCES = sorted(CSRC.glob("*.cu"))


def _behind(text, at, opening, closing):
    """The place behind the bracket that closes the one at ``at``."""
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == opening) - (text[i] == closing)
        if depth == 0:
            return i + 1
    raise AssertionError("unbalanced")


def _functions(text):
    """(name, whether it is a kernel, parameters, body) of the device functions of a source."""
    text = re.sub(r"//[^\n]*", "", text)
    out = []
    for m in re.finditer(r"__(global|device)__\s", text):
        head = re.compile(r"(?:__launch_bounds__\s*\([^{;]*?\)\s*)?(?:[\w:<>&*\s]|__\w+__)*?\b(\w+)\s*\(")
        at = m.end()
        bounds = re.compile(r"[^({;]*__launch_bounds__\s*\(").match(text, at)
        if bounds:
            at = _behind(text, bounds.end() - 1, "(", ")")
        h = head.match(text, at)
        if h is None:
            continue
        end = _behind(text, h.end() - 1, "(", ")")
        rest = re.match(r"\s*(?:const\s*)?\{", text[end:])
        if rest is None:
            continue
        brace = end + rest.end() - 1
        out.append((h.group(1), m.group(1) == "global", text[h.end():end - 1], text[brace:_behind(text, brace, "{", "}")]))
    return out


def _waits(body):
    """What the waits of a body take."""
    return [a.strip() for args in re.findall(r"\bgrid_(?:wait|begin)\(([^()]*)\)", body) for a in args.split(",") if a.strip()]


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_constant_reads_are_behind_the_wait(source):
    functions = _functions(source.read_text())
    bodies = {}
    for name, _kernel, _params, body in functions:
        bodies.setdefault(name, []).append(body)

    def reached(body, seen):
        """Bodies of the functions that one calls."""
        out = [body]
        for name in set(re.findall(r"\b(\w+)\s*(?:<[^;(){}]*>)?\s*\(", body)) & set(bodies) - seen:
            seen.add(name)
            for b in bodies[name]:
                out += reached(b, seen)
        return out

    for name, kernel, params, body in functions:
        if not kernel:
            continue
        parts = reached(body, {name})
        if not any(re.search(r"\bgrid_(wait|begin)\(", b) for b in parts):
            continue                             # launched behind all of the one before
        taken = [a for b in parts for a in _waits(b)]
        if any(re.search(r"\b__ldg\(", b) for b in parts):
            assert taken, f"{source.name}: {name} reads by __ldg, its wait takes no pointer"
        for p in params.split(","):
            m = re.search(r"\bconst\b[^,]*\*\s*__restrict__\s+(\w+)", p)
            if m:
                assert m.group(1) in taken, f"{source.name}: {name} reads {m.group(1)}, which its wait does not take"


def test_all_kernels_are_looked_at():
    """As many kernels as the sources say there are."""
    for source in SOURCES:
        text = re.sub(r"//[^\n]*", "", source.read_text())
        assert sum(k for _n, k, _p, _b in _functions(text)) == len(re.findall(r"\b__global__\b", text)), source.name
