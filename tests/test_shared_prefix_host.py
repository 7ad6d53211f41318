"""decode_shared's host side on the CPU: the shared length, refusals of the Python call and of the C entry."""

import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

import numpy as np
import pytest
import torch

from lvattn import Context, MI355XAttention, _capi, checks, shared_prefix_len


def test_shared_prefix_len():
    head = [9, 4, 7, 1]
    lists = [head + [2, 3], head + [5], head + [6, 8, 10]]
    assert shared_prefix_len(lists, [90, 70, 100], 16) == 64
    assert shared_prefix_len(lists, [90, 63, 100], 16) == 48  # a row whose cached keys end inside the fourth page
    assert shared_prefix_len(lists, [90, 15, 100], 16) == 0
    assert shared_prefix_len([head, head], [64, 64], 16) == 64
    assert shared_prefix_len([head, head[:2]], [64, 32], 16) == 32
    assert shared_prefix_len([head, [4] + head[1:]], [64, 64], 16) == 0  # the first page differs
    assert shared_prefix_len([head, head[:3] + [2]], [64, 64], 16) == 48
    assert shared_prefix_len([head, []], [64, 0], 16) == 0
    assert shared_prefix_len([head], [64], 16) == 0 and shared_prefix_len([], [], 16) == 0
    got = shared_prefix_len([np.array(head), tuple(head)], np.array([64, 64]), 16)
    assert got == 64 and type(got) is int
    for n in range(12):  # against the definition, over lengths
        a, b = list(range(12)), list(range(n)) + [99] * (12 - n)
        assert shared_prefix_len([a, b, a], [12 * 8] * 3, 8) == 8 * n
    with pytest.raises(ValueError, match="2 block lists for 1 rows"):
        shared_prefix_len([head, head], [64], 16)


def test_common_blocks_under_every_kind_of_row():
    from lvattn import _hoststage as hs

    assert hs.common_blocks([]) == 0 and hs.common_blocks([[]]) == 0 and hs.common_blocks([[5, 6]]) == 2
    assert hs.common_blocks([(1, 2, 3), np.array([1, 2, 4]), [1, 2]]) == 2
    assert hs.common_blocks([[1, 2], [], [1, 2]]) == 0
    for bad in (3, [[1], 3], [["a"], [1]], [[1], ["a"]], [[1 << 70], [1]]):
        with pytest.raises((TypeError, OverflowError)):
            hs.common_blocks(bad)


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_common_blocks_under_the_address_sanitizer(tmp_path):
    """The program of test_host_asan.py, driving common_blocks over ragged lists of every kind."""
    from test_host_asan import DRIVER, SOURCE

    libdir, ldver = sysconfig.get_config_var("LIBDIR"), sysconfig.get_config_var("LDVERSION")
    if not (Path(libdir) / f"libpython{ldver}.so").exists():
        pytest.skip("no shared libpython to embed")
    (tmp_path / "driver.cpp").write_text(DRIVER)
    (tmp_path / "script.py").write_text(SCRIPT)
    exe = tmp_path / "common"
    build = subprocess.run(
        ["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", f"-I{sysconfig.get_paths()['include']}",
         str(SOURCE), str(tmp_path / "driver.cpp"), f"-L{libdir}", f"-lpython{ldver}", f"-Wl,-rpath,{libdir}", "-o",
         str(exe)], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    env = {"ASAN_OPTIONS": "detect_leaks=0:halt_on_error=1", "UBSAN_OPTIONS": "halt_on_error=1",
           "PYTHONHOME": sys.base_prefix, "PATH": "/usr/bin:/bin"}
    run = subprocess.run([str(exe), str(tmp_path / "script.py")], capture_output=True, text=True, env=env, timeout=300)
    assert run.returncode == 0 and "common ok" in run.stdout, run.stdout[-2000:] + run.stderr[-4000:]


SCRIPT = """
import random
import _hoststage as hs
import numpy as np
rng = random.Random(0)
for trial in range(2000):
    head = [rng.randint(0, 1 << 31) for _ in range(rng.randint(0, 20))]
    rows = []
    for r in range(rng.randint(1, 8)):
        ids = head[:rng.randint(0, len(head))] + [rng.randint(0, 3) for _ in range(rng.randint(0, 4))]
        rows.append([list, tuple, lambda x: np.asarray(x, dtype=np.int64)][rng.randrange(3)](ids))
    want = 0
    while all(len(x) > want for x in rows) and len({int(x[want]) for x in rows}) == 1:
        want += 1
    assert hs.common_blocks(rows) == want, (rows, want)
    assert hs.common_blocks(tuple(rows)) == want
    try:
        hs.common_blocks(rows[:1] + [7] + rows)
        assert len(rows[0]) == 0
    except TypeError:
        pass
print("common ok")
"""


BF = torch.bfloat16


def args(q=(4, 8, 64), cache=(10, 16, 2, 64), tables=(4, 6), lens=4, dtype=BF, cache_dtype=BF, table_dtype=torch.int32):
    kc = torch.zeros(cache, dtype=cache_dtype)
    return dict(q=torch.zeros(q, dtype=dtype), k_cache=kc, v_cache=kc.clone(),
                context=Context(context_lens=torch.ones(lens, dtype=torch.int32),
                                block_tables=torch.zeros(tables, dtype=table_dtype)), shared_len=32)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=torch.float32), "not bf16 or fp16"), (dict(q=(4, 6, 64)), "q is"), (dict(q=(4, 8, 128)), "q is"),
    (dict(cache=(10, 16, 4, 64)), "caches"), (dict(cache=(64,)), "caches"), (dict(cache_dtype=torch.float16), "caches"),
    (dict(q=(5, 8, 64)), "do not divide"), (dict(lens=0, tables=(0, 6)), "do not divide"),
    (dict(tables=(3, 6)), "block tables"), (dict(table_dtype=torch.int64), "block tables"),
    (dict(tables=(4, 1)), "32 shared keys are not whole pages of 16 within tables of 1"), (dict(), "on one GPU"),
])
def test_the_call_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        MI355XAttention(8, 64, 0.125, 2).decode_shared(**args(**change))


def test_the_call_refuses_lengths_and_outputs():
    backend, a = MI355XAttention(8, 64, 0.125, 2), args()
    for bad in (-16, 8, 112):
        with pytest.raises(ValueError, match=f"{bad} shared keys"):
            backend.decode_shared(**(a | dict(shared_len=bad)))
    for out in (torch.zeros(4, 8, 128, dtype=BF), torch.zeros(1, 8, 64, dtype=BF).expand(4, 8, 64)):
        with pytest.raises(ValueError, match="out is"):
            backend.decode_shared(**a, out=out)
    for context in (Context(), Context(block_tables=a["context"].block_tables),
                    Context(block_tables=torch.zeros(4, dtype=torch.int32), context_lens=a["context"].context_lens)):
        with pytest.raises(ValueError, match="no block tables"):
            backend.decode_shared(**(a | dict(context=context)))


def test_the_debug_check_finds_pages_that_are_not_shared():
    tables, lens = torch.tensor([[3, 4, 5], [3, 9, 6], [3, 4, -1]]), torch.tensor([40, 40, 33])
    checks.check_shared(tables, lens, 1, 16, 1)
    with pytest.raises(ValueError, match="row 1's first 2 pages are not row 0's"):
        checks.check_shared(tables, lens, 2, 16, 1)
    lens[1] = 20  # does not see both pages: its own table counts
    checks.check_shared(tables, lens, 2, 16, 1)
    with pytest.raises(ValueError, match="row 0's"):
        checks.check_shared(torch.full((2, 3), -1), lens[:2], 1, 16, 1)


def c_call(*, rows=4, queries=1, hq=8, hk=2, dim=64, page=16, shared=32, max_k=96, scale=0.1, ws=16, nbytes=1 << 40,
           dtype=0, q=16, stride=64):
    _capi.call("lv_shared_prefix_decode", q, 8 * 64, stride, 16, 16, 2048, 128, 64, page, 16, 6, 16, rows, queries, hq, hk,
               dim, scale, shared, max_k, 0, 16, 512, 64, ws, nbytes, dtype, None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=3), "not bf16 or fp16"), (dict(rows=-1), "bad sizes"), (dict(queries=0), "bad sizes"),
    (dict(hq=9), "do not group"), (dict(dim=96), "head_dim 96"), (dict(queries=17), "17 queries of 4 heads"),
    (dict(page=24, shared=24), "page size 24"), (dict(page=0), "page size 0"), (dict(max_k=-1, shared=0), "max_seqlen_k"),
    (dict(max_k=(1 << 30) + 1), "above 2\\^30"), (dict(shared=40), "40 shared keys"), (dict(shared=-16), "-16 shared"),
    (dict(shared=112), "112 shared keys"), (dict(rows=1 << 26), "more than one launch holds"), (dict(q=None), "null"),
    (dict(q=18), "16-byte aligned"), (dict(stride=4), "16-byte aligned"), (dict(scale=0.0), "scale must be positive"),
    (dict(ws=None), "workspace of"), (dict(nbytes=64), "workspace of 64 bytes given"), (dict(ws=48), "256-byte aligned"),
])
def test_the_c_entry_refuses(change, message):
    with pytest.raises(_capi.LvError, match=message):
        c_call(**change)


def test_no_rows_and_the_workspace():
    c_call(rows=0)

    def size(*a, own_keys=0):
        return _capi.query("lv_shared_prefix_workspace_bytes", *a, own_keys)

    assert size(0, 1, 8, 2, 64, 16, 32, 96) == 0 and size(4, 1, 8, 3, 64, 16, 32, 96) == 0
    assert 0 < size(4, 1, 16, 8, 128, 16, 2048, 4096) < 8 << 20
    # at any length of context and batch a share of what its rows' caches take
    for rows in (1, 16, 256, 2048):
        for shared in (0, 4096, 1 << 20):
            assert size(rows, 1, 32, 8, 128, 256, shared, 1 << 21) < 400 << 20
