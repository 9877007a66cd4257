"""The chunk planner and the engine's speculative bookkeeping at their edges. No GPU needed."""
import numpy as np
import pytest
import torch

import deserve_b200 as dk
from deserve_b200 import _lib, ops


def _plan(new, pages, hq=64, hkv=8, d=128, ps=16, dtype=torch.bfloat16, workspace_bytes=None, capacity=None):
    qo, kv = (np.concatenate([[0], np.cumsum(v)]).astype(np.int32) for v in (new, pages))
    plan = np.zeros(ops.chunk_plan_capacity(int(qo[-1]), len(new)) if capacity is None else capacity, dtype=np.int32)
    used, ws = ops.make_chunk_plan(qo, kv, hq, hkv, d, ps, dtype, 148, plan, workspace_bytes)
    return plan[:used], ws


def _check_cover(plan, new, pages):
    """Every (row, page) once: rows of an item see the pages [first, end) of their request."""
    seen = [np.zeros((n, p), dtype=int) for n, p in zip(new, pages)]
    for req, q0, nq, pb, pe, *_ in plan[16: 16 + 12 * plan[1]].reshape(-1, 12):
        seen[req][q0: q0 + nq, pb:pe] += 1
    for s, p in zip(seen, pages):
        assert (s <= 1).all() and (s[-1] == 1).all()  # (pages behind a tile may be left out, the last row sees all)


BIG = [([64] * 8, [131072 // 16] * 8), ([512] * 4, [2048] * 4), ([1024], [8192]), ([5], [4096]), ([3, 1, 40], [9000, 2, 600])]


@pytest.mark.parametrize("new,pages", BIG)
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 128), (torch.float16, 96)])
@pytest.mark.parametrize("room", [127 << 20, 1 << 20, 5000, 0])
def test_chunk_plan_splits_no_further_than_its_workspace(new, pages, dtype, d, room):
    free, wanted = _plan(new, pages, dtype=dtype, d=d)
    plan, ws = _plan(new, pages, dtype=dtype, d=d, workspace_bytes=room)
    assert ws <= room and ws == plan[10] * 64 * (d + 2) * 4
    _check_cover(plan, new, pages)
    if wanted <= room:
        assert np.array_equal(plan, free)


def test_chunk_plan_splits_no_further_than_its_plan_holds():
    new, pages = [40, 5], [4096, 3000]
    free, _ = _plan(new, pages, dtype=torch.float32)
    plan, ws = _plan(new, pages, dtype=torch.float32, workspace_bytes=0)
    less, _ = _plan(new, pages, dtype=torch.float32, capacity=len(plan))  # unsplit tiles just fit
    assert len(free) > len(plan) and ws == 0 and len(less) <= len(plan)
    _check_cover(less, new, pages)
    with pytest.raises(_lib.DeserveKVError, match="plan needs"):
        _plan(new, pages, dtype=torch.float32, capacity=len(plan) - 1)
    with pytest.raises(ValueError, match="workspace_capacity"):
        _plan(new, pages, workspace_bytes=-1)


def test_chunk_plan_keeps_positions_within_32_bits():
    """Kernels walk a request in steps of a tile: the step behind its last token has to be a 32-bit position too."""
    for pages in ((1 << 27) - 1, (1 << 27) - 63):
        with pytest.raises(ValueError, match="2\\^31"):
            _plan([1], [pages])
    plan, _ = _plan([1], [(1 << 27) - 64])
    _check_cover_ends(plan, (1 << 27) - 64)


def _check_cover_ends(plan, pages):
    items = sorted(tuple(it[3:5]) for it in plan[16: 16 + 12 * plan[1]].reshape(-1, 12))
    assert items[0][0] == 0 and items[-1][1] == pages and all(a[1] == b[0] for a, b in zip(items, items[1:]))


BEYOND_MEMORY = """
import ctypes, resource
import numpy as np
from deserve_b200 import _lib
size = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (size + (64 << 20),) * 2)
qo, kv = np.array([0, 2**31 - 1], dtype=np.int32), np.array([0, 1], dtype=np.int32)
plan, used, ws = np.zeros(4096, dtype=np.int32), ctypes.c_int64(), ctypes.c_int64()
for capacity in (4096, 2**62):  # what there is, and more than the planner can have
    rc = _lib.lib.dsv_chunk_plan(qo.ctypes.data, kv.ctypes.data, 1, 1, 1, 64, 16, _lib.dtype_code(__import__("torch").float32), 148,
                                 plan.ctypes.data, capacity, ctypes.byref(used), ctypes.byref(ws))
    assert rc == _lib.E_WORKSPACE, rc
    print(_lib.last_error())
"""


def test_chunk_plan_beyond_memory_is_an_error_code():
    """2^31 - 1 new tokens, 64 MiB left to the process: refused by the capacity, or by the allocation that fails; not the end of the
    process."""
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-c", BEYOND_MEMORY], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    needs, alloc = r.stdout.splitlines()[-2:]
    assert "plan needs" in needs and "alloc" in alloc


def test_sample_top_p_does_not_write_probabilities_over_its_logits():
    buf = np.zeros(256, dtype=np.float32)
    at = buf.ctypes.data
    assert _lib.lib.dsv_sample_top_p(at, 64, 2, 64, at, at, at, at, at, 64, _lib.dtype_code(torch.float32), None) == _lib.E_INVALID
    assert "must not be logits" in _lib.last_error()


# ---- stages and tasks ------------------------------------------------------------------------------------------------------------
ARGS = dk.ModelArgs(dim=64, n_layers=2, n_heads=2, n_kv_heads=1, vocab_size=64, ffn_dim=64)


def test_a_split_head_does_not_sample():
    with pytest.raises(ValueError, match="split head is greedy"):
        dk.LlamaStage(ARGS, 0, 2, "cpu", torch.float32, split_head=True, sample_seed=1)
    assert dk.LlamaStage(ARGS, 0, 2, "cpu", torch.float32, sample_seed=1).generator is not None
    assert dk.LlamaStage(ARGS, 0, 2, "cpu", torch.float32, split_head=True).generator is None


@pytest.mark.parametrize("layers", [(0, 1), (1, 2), (0, 2)])
def test_a_split_head_does_not_verify(layers):
    """Refused before the caches grow."""
    stage = dk.LlamaStage(ARGS, *layers, "cpu", torch.float32, split_head=True)
    task = dk.TaskData.empty("a", 0)
    task.init(3)
    batch = dk.BatchVerify(torch.zeros(3, dtype=torch.int32), stage, [task], [None])
    with pytest.raises(ValueError, match="split head"):
        batch.prepare()


@pytest.mark.parametrize("fed,accepted,max_new,max_len,start,moved,left", [
    (5, 4, 100, 1000, 50, 5, 95),   # no limit near
    (5, 4, 5, 1000, 50, 5, 0),      # the limit met exactly
    (5, 4, 3, 1000, 50, 3, 0),      # two tokens too many
    (5, 4, 1, 1000, 50, 1, 0),
    (5, 2, 100, 52, 50, 2, 98),     # the length limit
    (5, 4, 100, 51, 50, 1, 99),
    (1, 0, 1, 1000, 50, 1, 0),      # no drafts
])
def test_commit_stops_at_the_limits_of_plain_decoding(fed, accepted, max_new, max_len, start, moved, left):
    plain = dk.TaskData.empty("p", start, dk.SamplingParams(max_new_tokens=max_new, max_seq_len=max_len))
    plain.start_pos, steps = start, 0
    while steps < accepted + 1:  # token by token, as LlamaStage.sample counts
        plain.init(1)
        plain.step()
        plain.sampling_params.max_new_tokens -= 1
        steps += 1
        if plain.sampling_params.max_new_tokens <= 0 or plain.start_pos >= max_len:
            break
    proc = dk.MicroBatchProcessor.__new__(dk.MicroBatchProcessor)
    proc.task_data_manager = dk.TaskManager(16, 16)
    task = dk.TaskData.empty("a", start, dk.SamplingParams(max_new_tokens=max_new, max_seq_len=max_len))
    proc.task_data_manager.add(task)
    task.start_pos = start
    task.init(fed)
    done = proc.commit(["a"], [accepted])
    assert (task.start_pos, task.sampling_params.max_new_tokens) == (plain.start_pos, plain.sampling_params.max_new_tokens) == (start + moved, left)
    assert done == (["a"] if left == 0 or start + moved >= max_len else [])
