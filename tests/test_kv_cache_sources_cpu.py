"""What of the cache kernels is shown by their sources: rules whose breach no run shows reliably."""
import re

from conftest import PKG_PARENT

CSRC = PKG_PARENT / "h3vae_b200" / "csrc"
SOURCES = [*sorted(CSRC.glob("kv_*.cu*")), *sorted(CSRC.glob("attention_kv*.cu*"))]


def _code(path):
    return re.sub(r"//[^\n]*", "", path.read_text())


def test_aligned_cluster_barriers_join_the_warp_first():
    """An .aligned barrier needs all lanes of a warp at once: each stands directly behind a __syncwarp()."""
    found = 0
    for path in SOURCES:
        lines = [x.strip() for x in _code(path).splitlines() if x.strip()]
        for before, line in zip(lines, lines[1:]):
            if "barrier.cluster" in line and ".aligned" in line:
                found += 1
                assert before == "__syncwarp();" and line.count("barrier.cluster") == 1, (path.name, line)
    assert found


def test_barriers_are_fenced_by_the_thread_that_initialised_them():
    """A fence after mbarrier.init orders the inits of its own thread: the statement that guards an init guards the
    fence too, and no second condition stands between them."""
    found = 0
    for path in SOURCES:
        code = _code(path)
        for match in re.finditer(r"mbar_init\((?:.|\n)*?fence_barrier_init\(\)", code):
            found += 1
            assert not re.search(r"\bif\s*\(", match.group(0)), path.name
        assert code.count("mbar_init(") == 0 or "fence_barrier_init()" in code, path.name
    assert found


def test_warps_stay_whole_around_loads_from_tensor_memory():
    """tcgen05.ld wants all lanes of a warp: a loop that loads does not let lanes go on to the next round by themselves."""
    code = _code(CSRC / "attention_kv_tile.cu")
    for call in re.finditer(r"\b(load_o|tmem_ld32|tmem_ld_wait)\(", code):
        body = code[call.end():]
        body = body[: min((body.find(x) for x in ("\n}", "#pragma unroll 1") if x in body), default=len(body))]
        assert "continue;" not in body, body[:200]


def test_nothing_throws_at_the_c_entries():
    """A C++ exception that leaves an extern "C" function ends the process: nothing that allocates or locks by throwing."""
    for path in SOURCES:
        code = _code(path)
        assert not re.search(r"std::(set|map|vector|string|function|mutex|lock_guard|unordered_\w+|call_once)\b", code), path.name
        assert not re.search(r"\b(throw|new)\b", code), path.name
