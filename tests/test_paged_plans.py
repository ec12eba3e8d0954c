"""What the rules of the paged cache's launches (csrc/paged_plan.h, csrc/weigh_plan.h: compiled here by g++) make of the
cases that the GPU tests were written for: a rule that changes must not take a test off the code that it is about."""
import ctypes
import os
import shutil
import subprocess

import pytest

from tests import test_gpu_paged_long as cases

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _compiled(tmp_path_factory, header, function):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    where = tmp_path_factory.mktemp("plan")
    (where / "plan.cpp").write_text(f'#include "{header}"\nextern "C" {function}\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "retrievalattention_amd", "csrc"),
                    str(where / "plan.cpp"), "-o", str(where / "plan.so")], check=True)
    return ctypes.CDLL(str(where / "plan.so")).ask


class Weigh(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("cols_pad", "S", "rows", "S2", "rows2", "per", "supers")] + [("joined", ctypes.c_bool),
                                                                                                       ("wide", ctypes.c_bool)]


@pytest.fixture(scope="module")
def weigh_plan(tmp_path_factory):
    call = _compiled(tmp_path_factory, "weigh_plan.h",
                     "void ask(long long groups, int cols, int T, WeighPlan* p) { *p = weigh_plan(groups, cols, T); }")

    def plan(groups, cols, T):
        p = Weigh()
        call(ctypes.c_longlong(groups), cols, T, ctypes.byref(p))
        return p
    return plan


def _walks(plan, second, cols, gs, W, T, lens):
    """(tiles of 64 keys, halves of a tile) of every workgroup's walk over a block of columns."""
    rows, block = (plan.rows2, 256 if plan.wide else 128) if second else (plan.rows, 256)
    walks = set()
    for n in lens:
        for c in range(0, cols, block):
            end = min(n, n - W + min(c + block - 1, cols - 1) // gs + 1)
            for j0 in range(0, T, rows):
                keys = min(j0 + rows, end) - j0
                if keys > 0:
                    walks.add((-(-keys // 64), -(-keys // 32)))
    return walks


def test_prompt_weights_stream_many_tiles(weigh_plan):
    """Both passes, of eight waves and of four, of 64 and 128 dims and either way of joining: walks of 1 to 6 tiles and of more, that end
    in either half of a tile."""
    walks, joined, supers = {}, set(), set()
    for _, heads, gs, dim, W, T, lens in cases.STREAMED:
        plan = weigh_plan(len(lens) * heads, W * gs, T)
        assert plan.per == 1 and plan.rows >= 7 * 64 and plan.rows2 >= 7 * 64
        joined.add(plan.joined)
        supers.add(min(plan.supers, 16))
        for key in ((dim, "first"), (dim, "wide" if plan.wide else "second")):
            walks.setdefault(key, set()).update(_walks(plan, key[1] != "first", W * gs, gs, W, T, lens))
    assert {1, 16} < supers and min(supers - {1}) < 16 and joined == {False, True}
    assert len(walks) == 6
    for key, seen in walks.items():
        tiles = {t for t, _ in seen}
        assert {1, 2, 3, 4, 5, 6} <= tiles and max(tiles) > 6, (key, sorted(tiles))
        assert {s % 2 for t, s in seen if t > 1} == {0, 1}, key


def test_prompt_weights_give_a_workgroup_several_blocks(weigh_plan):
    """Two and three, with fewer left for the last one, and blocks that begin in front of the prompt or see none of a split."""
    plans = {}
    for _, heads, gs, dim, W, T, lens, _ in cases.BLOCKS:
        plan = weigh_plan(len(lens) * heads, W * gs, T)
        blocks = -(-W * gs // 128)
        assert plan.per > 1 and plan.supers > 1 and plan.supers == -(-blocks // plan.per)
        plans[plan.per] = (blocks % plan.per != 0) or plans.get(plan.per, False)
    assert plans == {2: True, 3: True}


@pytest.fixture(scope="module")
def shares(tmp_path_factory):
    """The workgroups that share a call's rows, and each one's place in the run: (workgroups, [(sequence, head, chunks)] of each)."""
    call = _compiled(tmp_path_factory, "paged_plan.h", """long long ask(long long groups, int max_len, long long total, int* workgroups) {
        *workgroups = paged_workgroups(groups, max_len); return *workgroups ? pg_each(total, *workgroups) : 0; }""")
    call.restype = ctypes.c_longlong

    def walk(heads, lens, starts=None, max_len=None):
        first = [min(s, n) for s, n in zip(starts or [0] * len(lens), lens)]
        chunks = [-(-n // 16) - s // 16 if s < n else 0 for s, n in zip(first, lens)]
        places = [c + 32 if c else 0 for c in chunks]      # (a group begins with 32 places without rows)
        total, workgroups = sum(places) * heads, ctypes.c_int()
        each = call(ctypes.c_longlong(heads * len(lens)), max_len or max(lens), ctypes.c_longlong(total), ctypes.byref(workgroups))
        if not workgroups.value:
            return 0, []
        runs, at = [[] for _ in range(workgroups.value)], 0
        for b, n in enumerate(places):
            for h in range(heads if n else 0):
                for i in range(at // each, -(-(at + n) // each)):
                    rows = min(at + n, (i + 1) * each) - max(at + 32, i * each)
                    if rows > 0:
                        runs[i].append((b, h, rows))
                at += n
        return workgroups.value, runs
    return walk


def test_attention_walks_past_the_first_table_entries(shares):
    """Waves that look at three and more batches of 64 table entries, with pages of every size, beginning in the middle too."""
    seen = {}
    for _, heads, gs, dim, page, lens, starts in cases.LONG:
        workgroups, runs = shares(heads, lens, starts)
        to_batch = 64 // (1 if page >= 16 else 16 // page)
        most = max(-(-chunks // 8) for run in runs for _, _, chunks in run)      # of a wave, eight to a workgroup
        assert workgroups == 512 and -(-most // to_batch) >= 3, (page, most)
        seen.setdefault(min(page, 16), set()).add(1 if gs <= 4 else 2 if gs <= 8 else 4)
    assert set(seen) == {1, 2, 4, 8, 16} and set().union(*seen.values()) == {1, 2, 4}


def test_attention_joins_many_parts(shares):
    """More than 64 to a group, up to all 512 that there are, and groups whose parts begin at a later workgroup."""
    most, later = [], False
    for _, heads, gs, dim, page, lens, starts in cases.PARTS:
        _, runs = shares(heads, lens, starts)
        of = {}
        for i, run in enumerate(runs):
            for b, h, _ in run:
                of.setdefault((b, h), []).append(i)
        most.append(max(len(p) for p in of.values()))
        later |= any(len(p) > 64 and p[0] > 0 for p in of.values())
    assert min(most) > 64 and max(most) > 448 and later and len({-(-m // 64) for m in most}) >= 3, most


def test_attention_shares_the_rows_of_more_sequences_than_threads(shares):
    for _, heads, gs, dim, page, room, B in cases.MANY:
        lens = cases._many_lengths(room, B)
        workgroups, runs = shares(heads, lens, [n // 3 if b % 2 else 0 for b, n in enumerate(lens)])
        assert B > 512 and workgroups > 0
        assert any(run and run[0][0] > 511 for run in runs) and any(run and run[0][0] < 512 for run in runs)
        if B > 1024:
            assert any(run and run[0][0] > 1023 for run in runs)
