"""Every wait of a kernel on a barrier ends by the clock: a poll of a phase that does not come
pauses for milliseconds, so that a count of polls alone is no limit (2^26 of them are days)."""
import pathlib
import re

CSRC = pathlib.Path(__file__).resolve().parents[1] / "cl-inference_b200" / "csrc"
FUNCTION = re.compile(r"__device__ __forceinline__ \w+ (\w+)\([^{;]*\{\n(.*?)\n\}\n", re.S)


def functions():
    for path in sorted(CSRC.glob("*.cu*")):
        for name, body in FUNCTION.findall(path.read_text()):
            yield path.name, name, body


def test_waits_are_bounded_by_time():
    seen = []
    for file, name, body in functions():
        if re.search(r"\b(for|while)\b", body) and re.search(r"\b(mbar_test|test|peek)\(", body):
            seen.append(name)
            assert "time_ns() - start" in body, (file, name)
    assert {"mbar_wait", "mbar_drain", "wait_spin", "mbar_wait_spin"} <= set(seen)


def test_polls_are_made_by_those_functions_alone():
    for path in sorted(CSRC.glob("*.cu*")):
        polls = sum(len(re.findall(r"mbarrier\.(?:try|test)_wait", body)) for file, _, body in functions() if file == path.name)
        assert polls == len(re.findall(r"mbarrier\.(?:try|test)_wait", path.read_text())), path.name
        calls = re.findall(r"(?:for|while) \([^\n]*(?:mbar_test|\btest)\(", path.read_text())
        assert len(calls) == sum(len(re.findall(r"(?:for|while) \([^\n]*(?:mbar_test|\btest)\(", body))
                                 for file, _, body in functions() if file == path.name), path.name
