"""What the speculative operators refuse, at the C ABI (before any launch) and in Python, and the chunk
planner. No GPU needed."""
import ctypes

import numpy as np
import pytest
import torch

import deserve_b200 as dk
from deserve_b200 import _lib, ops

BUF = (ctypes.c_char * 4096)()
AT = (ctypes.addressof(BUF) + 63) // 64 * 64


def _plan(new, pages, hq=32, hkv=8, d=128, ps=16, dtype=torch.bfloat16, sms=148):
    qo = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    kv = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    plan = np.zeros(ops.chunk_plan_capacity(int(qo[-1]), len(new), sms), dtype=np.int32)
    used, ws = ops.make_chunk_plan(qo, kv, hq, hkv, d, ps, dtype, sms, plan)
    return plan[:used], ws, qo


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,ps", [(32, 8, 128, 16), (64, 8, 128, 16), (8, 2, 64, 16), (24, 1, 64, 16), (6, 3, 128, 5),
                                         (300, 1, 128, 16)])
@pytest.mark.parametrize("new,pages", [([1] * 200, [3] * 200), ([5], [4096]), ([1, 0, 33, 7, 2], [100, 50, 3, 0, 1]),
                                       ([257, 100], [300, 17]), ([3] * 1000, [1] * 1000), ([], []), ([0, 0], [4, 0])])
def test_chunk_plan_covers_every_row_and_page_once(dtype, hq, hkv, d, ps, new, pages):
    plan, ws, qo = _plan(new, pages, hq, hkv, d, ps, dtype)
    n_items, n_merge, tile, batch, parts_total = plan[1], plan[2], plan[3], plan[4], plan[10]
    assert batch == len(new) and plan[5] == 16 and plan[6] == 16 + 12 * n_items and len(plan) == plan[6] + 4 * n_merge
    assert ws == parts_total * hq * (d + 2) * 4 and plan[13] == qo[-1]
    items = plan[16: 16 + 12 * n_items].reshape(-1, 12)
    merge = {int(m[0]): m[1:].tolist() for m in plan[plan[6]:].reshape(-1, 4)}
    assert len(merge) == n_merge
    cover = [np.zeros((n, p), dtype=int) for n, p in zip(new, pages)]
    rows = [np.zeros(n, dtype=int) for n in new]
    part = np.zeros(parts_total, dtype=int)
    for req, q0, nq, pb, pe, slot, row, first, n_pages, left, *_ in items:
        assert row == qo[req] + q0 and left == new[req] - q0 and n_pages == pages[req] and first == sum(pages[:req])
        assert 0 <= q0 and 1 <= nq <= tile and q0 + nq <= new[req] and 0 <= pb <= pe <= pages[req]
        cover[req][q0: q0 + nq, pb:pe] += 1
        rows[req][q0: q0 + nq] += 1
        for j in range(nq):
            at = int(qo[req]) + q0 + j
            if slot < 0:
                assert at not in merge
                continue
            first, parts, step = merge[at]
            k, rest = divmod(slot + j - first, step)
            assert rest == 0 and 0 <= k < parts and step == nq
            part[slot + j] += 1
    assert (part == 1).all()
    for i, (n, p) in enumerate(zip(new, pages)):
        for j in range(n):
            at = int(qo[i]) + j
            assert rows[i][j] == (merge[at][1] if at in merge else 1)
            # every page that the row can see is read once; pages behind the tile may be left out
            seen = min(p, max(0, -(-(p * ps - n + j + 1) // ps)))
            assert (cover[i][j, :seen] == 1).all() and (cover[i][j] <= 1).all()


def test_chunk_plan_spreads_one_request_over_the_gpu():
    plan, _, _ = _plan([5], [4096])
    assert 140 <= plan[1] * 8 <= 592  # one CTA per item and kv head: about one round of the 148 SMs, at most four
    plan, ws, _ = _plan([4] * 600, [40] * 600)
    assert ws == 0  # enough requests: nothing is split


def test_chunk_plan_refusals():
    for kw, msg in (({"hq": 30}, "multiple"), ({"d": 100}, "head_dim"), ({"d": 264}, "head_dim"), ({"ps": 0}, "page_size"),
                    ({"dtype": torch.int32}, "dtype")):
        with pytest.raises(ValueError, match=msg):
            _plan([3, 1], [4, 5], **kw)
    with pytest.raises(ValueError, match="monotone"):
        _plan([3, -1], [4, 5])
    with pytest.raises(ValueError, match="monotone"):
        _plan([3, 1], [4, -5])
    with pytest.raises(ValueError, match="2\\^31"):
        _plan([3], [1 << 28])
    small = np.zeros(8, dtype=np.int32)
    with pytest.raises(_lib.DeserveKVError, match="plan needs"):
        ops.make_chunk_plan(np.array([0, 3]), np.array([0, 9]), 8, 2, 64, 16, torch.float32, 148, small)
    with pytest.raises(ValueError, match="batch"):
        ops.make_chunk_plan(np.array([0, 3]), np.array([0, 9, 12]), 8, 2, 64, 16, torch.float32, 148, small)


SMALL_PLAN, _, _ = _plan([2], [3], 8, 2, 64)


def _chunk_args(**kw):
    plan = SMALL_PLAN
    a = dict(q=AT, q_stride=512, qo=AT, pages=AT, page_stride=4096, num_pages=4, idx=AT, indptr=AT, last=AT, out=AT, out_stride=512,
             lse=None, plan=plan.ctypes.data, plan_dev=AT, ws=None, ws_bytes=0, batch=1, nnz=2, hq=8, hkv=2, d=64, ps=16, dtype=2,
             scale=0.1, stream=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,message", [
    ({"q": None}, "null pointer"), ({"plan": None}, "null pointer"), ({"idx": None}, "null pointer"), ({"dtype": 7}, "dtype"),
    ({"nnz": -1}, "negative"), ({"hq": 7}, "head counts"), ({"d": 60}, "head_dim"), ({"ps": 0}, "page_size"), ({"num_pages": 0}, "num_pages"),
    ({"batch": 2}, "does not belong"), ({"hkv": 4}, "does not belong"), ({"dtype": 0}, "does not belong"), ({"ps": 8}, "does not belong"),
    ({"nnz": 1}, "covers 2 rows"), ({"q": AT + 8}, "aligned"), ({"q_stride": 513}, "aligned"), ({"q_stride": 256}, "smaller than a row"),
    ({"page_stride": 2048}, "smaller than one page"), ({"plan_dev": AT + 4}, "aligned"),
])
def test_chunk_attention_refuses(kw, message):
    a = _chunk_args(**kw)
    assert _lib.lib.dsv_paged_chunk_attention(*a.values()) == _lib.E_INVALID
    assert message in _lib.last_error()


def test_chunk_attention_refuses_a_small_workspace_and_ignores_empty_calls():
    plan, ws, _ = _plan([2], [4000], 8, 2, 64)
    assert ws > 0
    a = _chunk_args(plan=plan.ctypes.data)
    assert _lib.lib.dsv_paged_chunk_attention(*a.values()) == _lib.E_WORKSPACE
    a["batch"] = 0
    assert _lib.lib.dsv_paged_chunk_attention(*a.values()) == 0
    a.update(batch=1, nnz=0)
    assert _lib.lib.dsv_paged_chunk_attention(*a.values()) == 0


@pytest.mark.parametrize("args,rc,message", [
    ((AT, 64, 2, 64, AT, AT, AT, AT, None, 0, 9, None), -1, "dtype"),
    ((AT, 64, -1, 64, AT, AT, AT, AT, None, 0, 2, None), -1, "bad shape"),
    ((AT, 64, 2, 0, AT, AT, AT, AT, None, 0, 2, None), -1, "bad shape"),
    ((AT, 1 << 19, 2, (1 << 18) + 1, AT, AT, AT, AT, None, 0, 2, None), -4, "vocabulary"),
    ((None, 64, 2, 64, AT, AT, AT, AT, None, 0, 2, None), -1, "null pointer"),
    ((AT, 64, 2, 64, None, AT, AT, AT, None, 0, 2, None), -1, "null pointer"),
    ((AT, 64, 2, 64, AT, AT, AT, None, None, 0, 2, None), -1, "null pointer"),
    ((AT, 63, 2, 64, AT, AT, AT, AT, None, 0, 2, None), -1, "smaller than a row"),
    ((AT, 64, 2, 64, AT, AT, AT, AT, AT, 63, 2, None), -1, "smaller than a row"),
    ((AT + 1, 64, 2, 64, AT, AT, AT, AT, None, 0, 2, None), -1, "misaligned"),
    ((None, 64, 0, 64, None, None, None, None, None, 0, 2, None), 0, ""),
])
def test_sample_top_p_refuses(args, rc, message):
    assert _lib.lib.dsv_sample_top_p(*args) == rc
    if rc:
        assert message in _lib.last_error()


def _verify_args(**kw):
    a = dict(logits=AT, stride=64, nnz=3, vocab=64, tokens=AT, indptr=AT, batch=1, u=AT, t=AT, k=AT, q=None, q_stride=0, ws=AT,
             ws_bytes=3, accepted=AT, following=AT, dtype=2, stream=None)
    a.update(kw)
    return a.values()


@pytest.mark.parametrize("kw,rc,message", [
    ({"dtype": 5}, -1, "dtype"), ({"nnz": -1}, -1, "bad shape"), ({"batch": -1}, -1, "bad shape"), ({"vocab": 0}, -1, "bad shape"),
    ({"vocab": 1 << 19, "stride": 1 << 19}, -4, "vocabulary"), ({"logits": None}, -1, "null pointer"), ({"tokens": None}, -1, "null pointer"),
    ({"indptr": None}, -1, "null pointer"), ({"ws": None}, -1, "null pointer"), ({"accepted": None}, -1, "null pointer"),
    ({"stride": 63}, -1, "smaller than a row"), ({"q": AT, "q_stride": 60}, -1, "smaller than a row"), ({"ws_bytes": 2}, -3, "workspace"),
    ({"logits": AT + 1}, -1, "misaligned"), ({"batch": 0}, 0, ""),
])
def test_verify_draft_refuses(kw, rc, message):
    assert _lib.lib.dsv_verify_draft(*_verify_args(**kw)) == rc
    if rc:
        assert message in _lib.last_error()


def test_operators_refuse_cpu_tensors():
    x, f = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        dk.sample_top_p(x, f, f, f)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        dk.verify_draft(x, torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), f, f[:1], f[:1])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        dk.paged_chunk_attention(torch.zeros(1, 2, 64), None, None, None, None, None, None, None, None)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        dk.BatchChunkWithPagedKVCacheWrapper(torch.zeros(4 << 20, dtype=torch.uint8))
