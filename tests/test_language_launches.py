"""What the operators of language models launch, written down by a program that answers for the device: sizes of the launches, what a failed one stops, and launches
that belong together."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "..", "dali_amd", "lib")


@pytest.fixture(scope="session")
def recorder(tmp_path_factory):
    program = str(tmp_path_factory.mktemp("recorder") / "launch_recorder")
    done = subprocess.run(["g++", "-std=c++17", "-O1", "-rdynamic", "-pthread", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-o", program, os.path.join(HERE, "launch_recorder.cpp"),
                           "-L" + LIB, "-ldali_hip", "-Wl,-rpath," + os.path.abspath(LIB), "-L/opt/rocm/lib", "-Wl,-rpath-link,/opt/rocm/lib"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert done.returncode == 0, done.stdout

    def run(*args):
        done = subprocess.run([program] + [str(a) for a in args], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
        assert done.returncode == 0, done.stdout
        return [line.split() for line in done.stdout.splitlines()]
    return run


ROWS = [1 << 16, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 24) - 1, 1 << 24, (1 << 24) + 5, 3 << 24]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", [0, 1])
def test_a_launch_has_fewer_than_2_to_32_threads(recorder, rows, dtype):
    for op, extents in (("log_probs", (8, 97, 1024, 2048, 2049, 8192, 50257)), ("log_probs_backward", (8, 97, 1024, 1025, 2049, 4096, 8191, 16384, 50257, 1 << 20)),
                        ("norm", (8, 97, 1024, 4096, 40000)), ("norm_backward", (8, 97, 1024, 4096, 40000))):
        for extent in extents:
            for k in (0, 5) if op == "log_probs" else (0,):
                (name, status, launches, blocks, threads), = recorder("one", op, dtype, rows, extent, k)
                assert int(status) == 0 and int(launches) >= 1 and int(threads) < 2 ** 32, (op, extent, k)


@pytest.mark.parametrize("op,extent", [("log_probs", 8), ("log_probs", 5000), ("log_probs_backward", 97), ("log_probs_backward", 20000)])
def test_a_failed_launch_is_the_last(recorder, op, extent):
    (_, status, launches, _, _), = recorder("one", op, 0, 5 << 24, extent, 0)
    assert int(status) == 0 and int(launches) > 2
    for failing in (0, 1):
        (_, status, launches, _, _), = recorder("one", op, 0, 5 << 24, extent, 0, failing)
        assert int(status) != 0 and int(launches) == failing + 1


@pytest.mark.parametrize("op,rows,extent", [("clip", 3, 100000), ("clip", 300, 100000), ("norm_backward", 5000, 1024), ("norm_backward", 5000, 40000)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_nothing_is_made_of_partial_sums_that_no_launch_left(recorder, op, rows, extent, dtype):
    (_, status, launches, _, _), = recorder("one", op, dtype, rows, extent, 0)
    assert int(status) == 0 and int(launches) > 1
    for failing in range(int(launches)):
        (_, status, made, _, _), = recorder("one", op, dtype, rows, extent, 0, failing)
        assert int(status) != 0 and int(made) == failing + 1


def test_a_call_without_memory_for_its_notes_fails(recorder):
    """An exception does not leave an entry of the library."""
    (status, *message), = recorder("memory")
    assert int(status) != 0 and "memory" in message


def test_two_threads_do_not_part_what_belongs_together(recorder):
    """The partial sums that one launch leaves are read by the next: what another thread launches between the two must not be such a pair's half."""
    assert [k for k, in recorder("threads", "squares")] == ["squares", "rescale", "norm_backward_team", "norm_fold"]
    assert [k for k, in recorder("threads", "norm_backward_team")] == ["norm_backward_team", "norm_fold", "squares", "rescale"]
    assert [k for k, in recorder("threads", "graph")] == ["graph_begins", "graph_ends", "squares", "rescale"]


def test_partial_sums_that_wait_for_another_launch_have_a_place_of_their_own(recorder):
    """Kernels that finish with the workspace within one launch may come between the two of a pair."""
    lines = recorder("places")
    assert all(int(status) == 0 for _, status, *_ in lines)
    places = {kind: sorted({int(p) for k, _, *found in lines if k == kind for p in found}) for kind in ("one", "two")}
    assert len(places["one"]) >= 2 and places["two"]
    partials = 65536 + (32 << 20)  # counters and the partial sums of single launches
    assert places["one"][-1] < partials <= places["two"][0]
