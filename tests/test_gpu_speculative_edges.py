"""Speculative operators where a border is met exactly, at the ends of the number range, and on calls that are allowed but
unusual. Expected tokens follow from the definition by counting: equal logits have equal weights, so running sums are whole
multiples of one weight and a dyadic random number meets a border exactly."""
import numpy as np
import pytest
import torch

import deserve_b200 as dk
from deserve_b200 import _lib, ops
from oracle import sampling as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.read_device_status() == 0, "a kernel self-check fired"


def _full(n, value):
    return torch.full((n,), float(value), device=DEV)


def _sample(row, rows, temperature, top_p, u, **kw):
    """Tokens of `rows` copies of one row."""
    x = row.to(DEV).expand(rows, -1).contiguous()
    return dk.sample_top_p(x, _full(rows, temperature), _full(rows, top_p), _full(rows, u), **kw).cpu()


def _last_row(row, requests, temperature, top_p, u):
    """The token that verification draws for requests without drafts."""
    x = row.to(DEV).expand(requests, -1).contiguous()
    n, tok = dk.verify_draft(x, torch.zeros(requests, dtype=torch.int32, device=DEV),
                             torch.arange(requests + 1, dtype=torch.int32, device=DEV), _full(requests, u),
                             _full(requests, temperature), _full(requests, top_p))
    assert (n == 0).all()
    return tok.cpu()


# ---- draws without a cut -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature,far", [(1.0, -32.0), (0.6, -20.0)])
@pytest.mark.parametrize("rows", [1, 128, 1024])
def test_a_draw_never_ends_among_weights_that_cannot_be_drawn(dtype, temperature, far, rows):
    """Two equal tokens, between them a vocabulary of weights below 2^-45 of theirs, no token at 0: a draw at one half meets
    the end of the first token's mass and takes the second."""
    row = torch.full((128256,), far, dtype=dtype)
    row[0], row[5000], row[128255] = -INF, 0.0, 0.0
    for draw in (_sample, _last_row):
        assert (draw(row, rows, temperature, 1.0, 0.5) == 128255).all()
        assert (draw(row, rows, temperature, 1.0, 0.5 - 2.0**-25) == 5000).all()


@pytest.mark.parametrize("vocab,value", [(1000, 0.0), (1000, 5.0), (5000, 5.0), (5000, -3.75), (4096, 0.3125), (32000, 7.5)])
@pytest.mark.parametrize("rows", [1, 40, 299, 1024])
def test_draws_at_exact_borders_do_not_depend_on_the_launch(vocab, value, rows):
    """All tokens equal: u of the whole is exactly the mass of the first u * vocab tokens, and the next one is drawn."""
    row = torch.full((vocab,), value)
    for u in (0.125, 0.25, 0.5, 0.75, 0.875):
        for draw in (_sample, _last_row):
            assert (draw(row, rows, 0.7, 1.0, u) == int(u * vocab)).all(), u


# ---- the nucleus' border -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,value", [(1000, 0.0), (1000, 0.3125), (1000, -3.75), (5000, 5.0), (32000, 7.5)])
@pytest.mark.parametrize("rows", [1, 40, 299, 1024])
def test_nucleus_borders_met_exactly_do_not_depend_on_the_launch(dtype, vocab, value, rows):
    """All tokens equal, top_p of the whole is exactly the mass of the first top_p * vocab tokens: the one behind them is kept too
    (the mass ranked before it is not more than top_p), and no other."""
    row = torch.full((vocab,), value, dtype=dtype)
    probs = torch.empty(rows, vocab, device=DEV)
    for top_p in (0.0, 0.125, 0.25, 0.5, 0.75):
        kept = int(top_p * vocab) + 1
        assert (_sample(row, rows, 0.7, top_p, 1 - 2.0**-24, probs=probs) == kept - 1).all()
        assert (probs[:, :kept] > 0).all() and (probs[:, kept:] == 0).all()
        assert (_last_row(row, rows, 0.7, top_p, 1 - 2.0**-24) == kept - 1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 128, 700])
def test_nucleus_borders_between_the_values_of_a_row(dtype, rows):
    """Eight tokens at the top, the other 1,016 entries at a 64th of their weight (their border lies behind the listed entries, or among
    them, depending on the launch): 8 + 1016 / 64 = 23.875 of the top's mass. top_p 0.5 keeps 11.9375 of it: 8 + 3.9375 * 64 = 252
    of the others rank before the border exactly, one more is kept."""
    row = torch.full((1024,), -6.0, dtype=dtype)
    row[500:508] = 0.0
    temperature = 1 / float(np.log(2.0))  # weights of 2^l; as fp32 off by up to 2^-25, the border by 6 * 2^-25 * 11 << 1 / 64
    probs = torch.empty(rows, 1024, device=DEV)
    _sample(row, rows, temperature, 0.5, 0.5, probs=probs)
    assert ((probs > 0).sum(1) - 8 - 252).abs().max() <= 1  # to the side on which the rounded temperature puts the border
    assert (probs == probs[0]).all()


# ---- the ends of the number range ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top_p", [0.9, 1.0])
@pytest.mark.parametrize("rest", ["ordinary", "masked", "lowest"])
def test_a_token_forced_by_the_largest_number_is_always_drawn(dtype, top_p, rest):
    info = torch.finfo(dtype)
    row = torch.randn(1000, generator=torch.Generator().manual_seed(1)) * 3
    row[::5] = -INF
    if rest != "ordinary":
        row[:] = -INF if rest == "masked" else info.min
    row[7], row[1:4] = info.max, torch.tensor([0.0, 1.0, -5.0])
    row = row.to(dtype)
    probs = torch.empty(3, 1000, device=DEV)
    for u in (0.0, 0.3, 0.999):
        for t in (1.0, 1e-3):
            assert (_sample(row, 3, t, top_p, u, probs=probs) == 7).all()
            assert (probs[:, 7] == 1).all() and probs.sum() == 3
            assert (_last_row(row, 3, t, top_p, u) == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_tokens_at_the_largest_number_share_a_row(dtype):
    row = torch.zeros(1000, dtype=dtype)
    row[7] = row[900] = torch.finfo(dtype).max
    for top_p in (0.9, 1.0):
        for u, want in ((0.25, 7), (0.5, 900), (0.75, 900)):
            assert (_sample(row, 2, 1.0, top_p, u) == want).all()
    assert (_sample(row, 2, 1.0, 0.25, 0.99) == 7).all()  # the nucleus ends with the first


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1e34, 1e36, 3e38, INF])
@pytest.mark.parametrize("hidden", [-INF, float("nan")])
def test_masked_entries_have_no_weight_at_any_temperature(dtype, temperature, hidden):
    """64 tokens among 131,072 entries, evenly likely: half of them side by side, half of them far apart."""
    at = list(range(100, 132)) + list(range(1000, 131072, 4096))
    row = torch.full((131072,), hidden, dtype=dtype)
    row[at] = torch.linspace(-3, 3, 64).to(dtype)
    for rows in (1, 300):
        for u in (0.0, 0.26, 0.51, 0.99):
            want = at[int(64 * u)]
            for top_p in (1.0, 1 - 2.0**-24):
                assert (_sample(row, rows, temperature, top_p, u) == want).all()
                assert (_last_row(row, rows, temperature, top_p, u) == want).all()


# ---- verification --------------------------------------------------------------------------------------------------------------
def _verify_one_draft(row, requests, draft, q, u, u_last, temperature=0.7, top_p=1.0):
    """Requests with one draft each, all alike: (accepted, next token) of every one."""
    x = row.to(DEV).expand(2 * requests, -1).contiguous()
    tokens = torch.full((2 * requests,), draft, dtype=torch.int32, device=DEV)
    uniform = torch.tensor([u, u_last], dtype=torch.float32, device=DEV).repeat(requests)
    indptr = torch.arange(0, 2 * requests + 1, 2, dtype=torch.int32, device=DEV)
    n, tok = dk.verify_draft(x, tokens, indptr, uniform, _full(requests, temperature), _full(requests, top_p),
                             None if q is None else q.to(DEV).expand(2 * requests, -1).contiguous())
    return n.cpu(), tok.cpu()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,value", [(1000, 5.0), (1024, 0.3125), (5000, -3.75), (32000, 7.5)])
@pytest.mark.parametrize("requests", [1, 40, 299, 700])
def test_residual_draws_at_exact_borders_do_not_depend_on_the_launch(dtype, vocab, value, requests):
    """The target is flat, the draft has all its mass on the first half: what is left is the second half, evenly."""
    q = torch.zeros(vocab)
    q[: vocab // 2] = 2 / vocab
    row = torch.full((vocab,), value, dtype=dtype)
    for u in (0.125, 0.25, 0.5, 0.75):
        n, tok = _verify_one_draft(row, requests, 3, q, 0.9, u)
        assert (n == 0).all() and (tok == vocab // 2 + int(u * (vocab // 2))).all()


@pytest.mark.parametrize("requests", [1, 40, 700])
def test_a_draft_whose_test_meets_equality_is_rejected(requests):
    """u q = p exactly is not u q < p; one step below it is accepted. The same under a nucleus that keeps every token."""
    row, q = torch.full((4096,), 0.3125), torch.zeros(4096)
    q[: 2048] = 2.0**-11
    for top_p in (1.0, 1 - 2.0**-24):
        for value in (row, row.to(torch.bfloat16)):
            assert (_verify_one_draft(value, requests, 3, q, 0.5, 0.5, top_p=top_p)[0] == 0).all()
            assert (_verify_one_draft(value, requests, 3, q, 0.5 - 2.0**-25, 0.5, top_p=top_p)[0] == 1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top_p", [0.9, 1.0])
def test_a_draft_that_cannot_be_drawn_is_rejected_by_every_random_number(dtype, top_p):
    row = torch.full((900,), -40.0, dtype=dtype)
    row[5] = row[700] = 0.0
    for draft, accepted in ((8, 0), (700, 1), (5, 1)):
        n, tok = _verify_one_draft(row, 2, draft, None, 0.0, 0.75, temperature=1.0, top_p=top_p)
        assert (n == accepted).all() and (tok == 700).all()
        n, tok = _verify_one_draft(row, 2, draft, torch.zeros(900), 0.3, 0.75, temperature=1.0, top_p=top_p)  # q(x) = 0
        assert (n == accepted).all() and (tok == 700).all()


# ---- calls that are refused on the device --------------------------------------------------------------------------------------
def test_verify_draft_with_an_indptr_that_is_not_monotone_reads_nothing_it_should_not():
    """Requests whose rows belong to no request of the search, drafts that are no tokens, and scratch full of old verdicts: the bad
    request is reported, the others end."""
    vocab, nnz = 5000, 8
    indptr = torch.tensor([0, 5, 3, 8], dtype=torch.int32, device=DEV)
    logits = torch.randn(nnz, vocab, generator=torch.Generator().manual_seed(1)).to(DEV)
    tokens = torch.full((nnz,), 2**31 - 1, dtype=torch.int32, device=DEV)
    tokens[1], tokens[4] = logits[0].argmax(), logits[3].argmax()
    u, one = _full(nnz, 1e-6), _full(3, 1.0)
    torch.cuda.synchronize()
    _lib.read_device_status()
    for old in (0x00, 0x01, 0x02):
        accepted, following = (torch.empty(3, dtype=torch.int32, device=DEV) for _ in range(2))
        scratch = torch.full((nnz,), old, dtype=torch.uint8, device=DEV)
        rc = _lib.lib.dsv_verify_draft(logits.data_ptr(), vocab, nnz, vocab, tokens.data_ptr(), indptr.data_ptr(), 3, u.data_ptr(),
                                       one.data_ptr(), one.data_ptr(), None, 0, scratch.data_ptr(), nnz, accepted.data_ptr(),
                                       following.data_ptr(), _lib.dtype_code(torch.float32), _lib.current_stream_ptr())
        assert rc == 0
        torch.cuda.synchronize()
        assert _lib.read_device_status() == 2  # inconsistent indptr
        assert (scratch <= 2).all() and following[1] == -1
        assert accepted.tolist() == [1, 0, 1]  # the last request gets to row 4, which the search gives to the first one
        assert ((following[[0, 2]] >= 0) & (following[[0, 2]] < vocab)).all()


# ---- chunk attention -----------------------------------------------------------------------------------------------------------
def _chunk_batch(seed, lens, new, hq, hkv, d, ps, dtype):
    """Requests over a shuffled pool: (wrapper, q, pages, page ids, first new row of every request)."""
    g = torch.Generator().manual_seed(seed)
    n_pages = [-(-n // ps) for n in lens]
    qo, kvp = (np.concatenate([[0], np.cumsum(v)]).astype(np.int32) for v in (new, n_pages))
    ids = torch.randperm(int(kvp[-1]) + 3, generator=g)[: int(kvp[-1])].to(torch.int32).to(DEV)
    pages = torch.randn(int(kvp[-1]) + 3, 2, ps, hkv, d, generator=g).to(dtype).to(DEV)
    q = torch.randn(int(qo[-1]), hq, d, generator=g).to(dtype).to(DEV)
    last = torch.tensor([(n - 1) % ps + 1 if n else 0 for n in lens], dtype=torch.int32, device=DEV)
    w = ops.BatchChunkWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device=DEV))
    w.begin_forward(torch.from_numpy(qo).to(DEV), torch.from_numpy(kvp).to(DEV), ids, last, hq, hkv, d, ps, dtype,
                    qo_indptr_host=qo, kv_indptr_host=kvp)
    return w, q, pages, ids, qo, kvp


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [INF, float("nan")])
@pytest.mark.parametrize("at", [0, 9, 31, 32, 50, 62])
def test_chunk_attention_with_two_q_tiles_finds_values_that_are_no_numbers(dtype, d, bad, at):
    """64 new tokens of 4 heads each, two q tiles that share their V: a new token's V that is no number reaches the rows from its own
    on, in both tiles, and no earlier one."""
    lens, new = [64, 700, 1290], [64, 64, 64]
    w, q, pages, ids, qo, kvp = _chunk_batch(at, lens, new, 8, 2, d, 16, dtype)
    clean = w.forward(q, pages)
    for i, n in enumerate(lens):
        t = n - 64 + at
        pages[int(ids[kvp[i] + t // 16]), 1, t % 16, :, 5] = bad
    for _ in range(10):
        got = w.forward(q, pages)
        for i in range(len(lens)):
            a = int(qo[i])
            assert torch.equal(got[a: a + at], clean[a: a + at])
            assert not torch.isfinite(got[a + at: a + 64, :, 5]).any()
            assert torch.isfinite(got[a + at: a + 64, :, :5]).all() and torch.isfinite(got[a + at: a + 64, :, 6:]).all()


@pytest.mark.parametrize("dtype,hq", [(torch.float32, 8), (torch.bfloat16, 8), (torch.bfloat16, 32)])
def test_chunk_attention_in_the_smallest_workspace(dtype, hq):
    """2 MiB: the plan of a batch that would be cut finer elsewhere; the same outputs up to rounding (each is within eps / 2 of the value
    plus eps / 2 of sum p |v| <= max |v| of the exact one, test_gpu_speculative.py)."""
    w, q, pages, ids, qo, kvp = _chunk_batch(3, [40000, 30000], [16, 9], hq, 2, 128, 16, dtype)
    want = w.forward(q, pages)
    small = ops.BatchChunkWithPagedKVCacheWrapper(torch.empty(2 << 20, dtype=torch.uint8, device=DEV))
    small.begin_forward(torch.from_numpy(qo).to(DEV), torch.from_numpy(kvp).to(DEV), ids,
                        torch.tensor([16, 16], dtype=torch.int32, device=DEV), hq, 2, 128, 16, dtype, qo_indptr_host=qo,
                        kv_indptr_host=kvp)
    assert small._plan_host[10] < w._plan_host[10]
    got = small.forward(q, pages)
    eps = torch.finfo(dtype).eps if dtype != torch.float32 else 2.0**-17
    assert ((got.float() - want.float()).abs() <= eps * (want.float().abs() + float(pages.abs().max()))).all()


@pytest.mark.parametrize("dtype,hq,lens,new", [(torch.bfloat16, 8, [5000, 33], [4, 3]), (torch.bfloat16, 8, [9000, 100], [40, 7]),
                                               (torch.float32, 4, [3000, 1], [2, 1])])
def test_functional_chunk_attention(dtype, hq, lens, new):
    """Every buffer explicit: the outputs of the wrapper with the same plan; buffers that the plan outgrows are refused."""
    hkv, d, ps = 2, 128, 16
    w, q, pages, ids, qo, kvp = _chunk_batch(7, lens, new, hq, hkv, d, ps, dtype)
    lse = torch.empty(q.shape[:2], device=DEV)
    want = w.forward(q, pages, lse=lse)
    plan = np.zeros(ops.chunk_plan_capacity(int(qo[-1]), len(new)), dtype=np.int32)
    used, ws_bytes = ops.make_chunk_plan(qo, kvp, hq, hkv, d, ps, dtype, _lib.device_info()[0], plan, 63 << 20)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    last = i32([(n - 1) % ps + 1 for n in lens])
    plan_dev, ws = torch.from_numpy(plan[:used]).to(DEV), torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=DEV)
    out, got_lse = torch.empty_like(q), torch.empty_like(lse)
    call = lambda **kw: dk.paged_chunk_attention(**{**dict(
        q=q, qo_indptr=i32(qo), paged_kv_cache=pages, kv_indices=ids, kv_indptr=i32(kvp), kv_last_page_len=last, plan_host=plan,
        plan_dev=plan_dev, workspace=ws, out=out, lse=got_lse), **kw})
    assert call() is out and torch.equal(out, want) and torch.equal(got_lse, lse)
    for kw, message in (({"kv_indices": ids[:-1]}, "kv_indices"), ({"plan_dev": plan_dev[:-1]}, "plan_dev"),
                        ({"plan_host": plan.astype(np.int64)}, "plan_host"), ({"plan_host": plan[:8]}, "plan_host"),
                        ({"out": out[:-1]}, "rows"), ({"lse": got_lse[:-1]}, "lse"), ({"kv_indptr": i32(kvp[:-1])}, "batch")):
        with pytest.raises(ValueError, match=message):
            call(**kw)
    if ws_bytes:
        with pytest.raises(_lib.DeserveKVError, match="workspace"):
            call(workspace=None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[3, 1], [40, 17]])
@pytest.mark.parametrize("scale", [0.0, -0.2, -3.0])
def test_chunk_attention_with_a_scale_that_is_not_positive(dtype, new, scale):
    """The definition holds for any scale. Tolerances as in test_gpu_speculative.py: a rounding of the result, one of each probability, fp32
    scores of 128 products."""
    w, q, pages, ids, qo, kvp = _chunk_batch(4, [900, 50], new, 8, 2, 128, 16, dtype)
    lse = torch.empty(q.shape[:2], device=DEV)
    out = w.forward(q, pages, sm_scale=scale, lse=lse)
    want, want_lse, size, reach = oracle.chunk_attention(q, pages, qo, ids, kvp, [900, 50], scale)
    eps = torch.finfo(dtype).eps if dtype != torch.float32 else 0.0
    arith = 2 * 130 * 2.0**-24 * reach + 2.0**-18
    tol = torch.finfo(dtype).eps / 2 * want.abs() + size * (eps / 2 + arith[..., None])
    assert ((out.double() - want).abs() <= tol).all()
    assert ((lse.double() - want_lse).abs() <= arith + 2.0**-23 * want_lse.abs()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[3], [2, 0, 40]])
def test_chunk_attention_of_a_batch_without_any_cache(dtype, new):
    """No request has a page: every row sees nothing."""
    w, q, pages, ids, qo, kvp = _chunk_batch(2, [0] * len(new), new, 8, 2, 128, 16, dtype)
    assert ids.numel() == 0
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 3.0, device=DEV)
    w.forward(q, pages, out=out, lse=lse)
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype,hq", [(torch.float32, 8), (torch.bfloat16, 8), (torch.float16, 32)])
def test_chunk_attention_reports_a_page_outside_the_pool(dtype, hq):
    """... and reads page 0 in its place; the requests that do not hold it are as before."""
    w, q, pages, ids, qo, kvp = _chunk_batch(5, [700, 90], [4, 3], hq, 2, 128, 16, dtype)
    want = w.forward(q, pages)
    for bad in (-1, len(pages), 2**31 - 1):
        kept = int(ids[7])
        ids[7] = bad
        got = w.forward(q, pages)
        torch.cuda.synchronize()
        assert _lib.read_device_status() == 1
        assert torch.equal(got[4:], want[4:]) and torch.isfinite(got).all()
        ids[7] = kept
