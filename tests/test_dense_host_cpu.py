"""The host side of the 8-bit product and the log probabilities over a runtime that stands in for the
device: which launches a call makes, what memory it takes, and that it does without where it can."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "objeta_amd", "lib")
STRAIGHTEN = (2048, 1, 256)


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("dense_host") / "check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "objeta_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "dense_host_check.cpp"), "-o", exe, "-rdynamic", "-L" + LIB, "-lobjeta_hip",
                    "-L/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath," + LIB, "-Wl,-rpath,/opt/rocm/lib"], check=True)

    def run(*commands):
        """Calls as (status, launches), and the sizes of the allocations."""
        out = subprocess.run([exe, *commands], capture_output=True, text=True, check=True, timeout=120).stdout.splitlines()
        calls = []
        for line in out[:-1]:
            status, *launches = line.split()
            calls.append((int(status), [tuple(map(int, x.split(","))) for x in launches]))
        return calls, [int(x) for x in out[-1].split()[1:]]
    return run


def test_product_without_memory_for_copies_reads_rows_where_they_lie(check):
    """Rows that begin anywhere are copied where there is room; without any the call computes the same
    from where they lie, as a captured one does."""
    (copied,), _ = check("product:1700,1650,37")
    assert copied[0] == 0 and copied[1][:2] == [STRAIGHTEN, STRAIGHTEN] and len(copied[1]) == 3
    (captured,), _ = check("capture:1", "product:1700,1650,37")
    assert captured[0] == 0 and len(captured[1]) == 1 and STRAIGHTEN not in captured[1]
    for room in (0, 16384, 100000):
        (short, again), _ = check(f"memory:{room}", "product:1700,1650,37", "product:1700,1650,37")
        assert short == captured and again == captured


def test_product_copies_stay_within_their_bounds(check):
    """Calls that climb in odd sizes: no region past 1 GiB, those it replaced together below another."""
    sizes, cols = [], 33
    while cols < 131071:
        sizes.append((2000, 2000, cols))
        cols = cols * 5 // 4 + 1 | 1
    sizes += [(2000 + 100 * i, 2000, 131071) for i in range(40)] + [(8190, 8192, 65535), (8192, 8192, 65535), (8192, 8192, 65535)]
    calls, regions = check(*(f"product:{n},{r},{k}" for n, r, k in sizes))
    for (n, r, k), (status, launches) in zip(sizes, calls):
        fits = (n + r) * ((k + 15) // 16 * 16) <= 1 << 30
        assert status == 0 and len(launches) == (3 if fits else 1), (n, r, k, launches)
    copies = regions[1:]  # (the first is the stream's own counters)
    assert max(copies) == copies[-1] <= 1 << 30 and sum(copies[:-1]) < 1 << 30, copies


@pytest.mark.parametrize("n,rows,cols,groups,threads", [
    (300, 14336, 4096, 112 * 2, 512),  # 128 x 256; 64 x 64 would be five tiles a CU in three rounds
    (8192, 28672, 1024, 112 * 32, 512),  # 256 x 256; 128 x 128 28 a CU in fourteen
    (2048, 32000, 256, 125 * 8, 512), (700, 32000, 5120, 125 * 3, 512), (20, 65536, 512, 512, 256),
    (15, 52105, 328, 815, 256),  # 64 x 64 of rows that begin anywhere: four share a CU
    (200, 160000, 256, 1250 * 2, 256),  # 128 x 128: 256 tokens a tile would be a fifth empty
    (512, 4096, 4096, 64 * 4, 256), (64, 14336, 4096, 224, 256), (64, 4096, 14336, 128 * 2, 512)])
def test_tiles_are_charged_for_every_round(check, n, rows, cols, groups, threads):
    """The tile of a product, of those that were timed, with what starts and ends it counted for every
    round of workgroups that the card takes in turn."""
    ((status, launches),), _ = check(f"product:{n},{rows},{cols}")
    assert status == 0 and launches == [((groups + 7) // 8 * 8, 1, threads)]


@pytest.mark.parametrize("rows,vocab,dtype", [(1, 151936, 0), (1, 200000, 0), (1, 262144, 0), (4, 262144, 0), (1, 1000000, 0), (1, 524288, 2),
                                              (3, 2000000, 2), (1, (1 << 31) - (1 << 16), 1)])
def test_the_join_holds_every_part_of_a_row(check, rows, vocab, dtype):
    """The best of a cut row are found from the largest value of each 64th of its parts, twenty held by each of
    256 threads; rows of which only sums are asked are cut as far as the join has threads."""
    (best, sums), _ = check(f"logprobs:{rows},{vocab},{dtype},20", f"logprobs:{rows},{vocab},{dtype},0")
    for (status, launches), most in ((best, 80), (sums, 256)):
        assert status == 0 and len(launches) == 2
        (n, parts, threads), join = launches
        assert n == rows and 1 < parts <= most and threads == 256 and join == (rows, 1, 256)
    assert sums[1][0][1] >= best[1][0][1]
