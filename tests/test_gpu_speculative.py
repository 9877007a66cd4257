"""Chunk attention, top-p sampling and draft verification on the GPU against their definitions in 64 bits.

Tokens and counts have to be equal. Attention outputs carry one rounding of the result (eps / 2 of its value), for 16-bit
types one of each probability (eps / 2 of it, so eps / 2 of A = sum p |v|), and fp32 arithmetic: a score of d products is off
by at most (d + 2) 2^-24 of B = sum |q k| scale, which moves every probability by twice that relatively; exp2 and the
running sums add a few units of 2^-24 (2^-18 covers 64 of them)."""
import numpy as np
import pytest
import torch

import deserve_b200 as dk
from deserve_b200 import _lib, ops
from oracle import sampling as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.read_device_status() == 0, "a kernel self-check fired"


# ---- chunk attention ---------------------------------------------------------------------------------------------------------
class Batch:
    """Requests of the given cache lengths and new tokens over a shuffled pool whose unused slots hold NaN."""

    def __init__(self, seed, lens, new, hq, hkv, d, ps, dtype, pool_stride=None, pad_rows=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.hq, self.hkv, self.d, self.ps, self.dtype = lens, new, hq, hkv, d, ps, dtype
        n_pages = [-(-n // ps) for n in lens]
        total = sum(n_pages)
        pool = total + total // 4 + 2
        self.qo = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.kvp = np.concatenate([[0], np.cumsum(n_pages)]).astype(np.int32)
        ids = torch.randperm(pool, generator=g)[:total].to(torch.int32)
        page = 2 * ps * hkv * d
        stride = page if pool_stride is None else pool_stride
        flat = torch.full((pool * stride,), float("nan"), dtype=dtype)
        pages = flat.as_strided((pool, 2, ps, hkv, d), (stride, ps * hkv * d, hkv * d, d, 1))
        for i, n in enumerate(lens):
            for j in range(n_pages[i]):
                k = min(ps, n - j * ps)
                pages[int(ids[self.kvp[i] + j]), :, :k] = torch.randn(2, k, hkv, d, generator=g).to(dtype)
        self.pages = flat.to(DEV).as_strided(pages.shape, pages.stride())
        self.ids = ids.to(DEV)
        self.last = torch.tensor([(n - 1) % ps + 1 if n else 0 for n in lens], dtype=torch.int32, device=DEV)
        self.q = torch.randn(int(self.qo[-1]) + pad_rows, hq, d, generator=g).to(dtype).to(DEV)
        self.qo_dev, self.kvp_dev = torch.from_numpy(self.qo).to(DEV), torch.from_numpy(self.kvp).to(DEV)
        self.wrapper = ops.BatchChunkWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device=DEV))

    def begin(self):
        self.wrapper.begin_forward(self.qo_dev, self.kvp_dev, self.ids, self.last, self.hq, self.hkv, self.d, self.ps, self.dtype,
                                   qo_indptr_host=self.qo, kv_indptr_host=self.kvp)
        return self

    def check(self, out, lse, scale=None):
        n = int(self.qo[-1])
        want, want_lse, size, reach = oracle.chunk_attention(self.q[:n], self.pages, self.qo, self.ids, self.kvp, self.lens, scale)
        eps = torch.finfo(self.dtype).eps if self.dtype != torch.float32 else 0.0
        arith = 2 * (self.d + 2) * 2.0**-24 * reach + 2.0**-18
        tol = torch.finfo(self.dtype).eps / 2 * want.abs() + size * (eps / 2 + arith[..., None])
        tiny = torch.finfo(self.dtype).smallest_normal
        err = (out[:n].double() - want).abs()
        assert (err <= tol + tiny).all(), float((err / (tol + tiny)).max())
        if lse is not None:
            seen = torch.isfinite(want_lse)
            assert torch.equal(torch.isneginf(lse[:n]), ~seen)
            err = (lse[:n].double() - want_lse).abs()[seen]
            assert (err <= (arith + 2.0**-23 * want_lse.abs())[seen]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,ps", [(32, 8, 128, 16), (8, 2, 64, 16), (64, 8, 128, 16), (4, 4, 64, 8), (5, 1, 128, 32),
                                         (10, 2, 96, 16), (24, 1, 64, 16), (2, 2, 256, 16), (6, 3, 128, 5), (12, 4, 8, 1)])
def test_chunk_attention_shapes(dtype, hq, hkv, d, ps):
    lens = [1, 2, ps, ps + 1, 3 * ps + 5, 700, 40, 257]
    new = [1, 2, 1, 3, 7, 5, 40, 17]
    b = Batch(hq * d + ps, lens, [min(n, m) for n, m in zip(new, lens)], hq, hkv, d, ps, dtype).begin()
    lse = torch.empty(b.q.shape[:2], device=DEV)
    out = b.wrapper.forward(b.q, b.pages, lse=lse)
    b.check(out, lse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("lens,new", [([20000], [1]), ([9001, 3, 5000], [5, 3, 16]), ([4097], [33]), ([300], [257])])
def test_chunk_attention_split_over_the_cache(dtype, hq, hkv, d, lens, new):
    b = Batch(3, lens, new, hq, hkv, d, 16, dtype).begin()
    lse = torch.empty(b.q.shape[:2], device=DEV)
    out = b.wrapper.forward(b.q, b.pages, lse=lse)
    b.check(out, lse)


@pytest.mark.parametrize("dtype", DTYPES)
def test_chunk_attention_rows_that_see_nothing_and_empty_requests(dtype):
    """More new tokens than cache (the first rows see nothing), a request without cache, one without new tokens."""
    b = Batch(5, [3, 0, 40, 17, 600], [5, 2, 0, 17, 1], 8, 2, 128, 16, dtype).begin()
    lse = torch.empty(b.q.shape[:2], device=DEV)
    out = b.wrapper.forward(b.q, b.pages, lse=lse)
    b.check(out, lse)
    assert (out[:2] == 0).all() and torch.isneginf(lse[:2]).all()
    assert (out[5:7] == 0).all() and torch.isneginf(lse[5:7]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_chunk_attention_strided_q_padded_rows_and_pool_gaps(dtype):
    """q as a column slice of a wider projection output, rows behind the last request left alone, a pool whose pages are
    farther apart than a page, an output with its own stride and scale."""
    hq, hkv, d, ps = 8, 2, 64, 16
    page = 2 * ps * hkv * d
    b = Batch(6, [100, 35, 900], [4, 1, 3], hq, hkv, d, ps, dtype, pool_stride=page + 64, pad_rows=5).begin()
    n = int(b.qo[-1])
    wide = torch.full((n + 5, 3, hq, d), 7.0, dtype=dtype, device=DEV)
    wide[:, 1] = b.q
    out = torch.full((n + 5, 2, hq, d), 3.0, dtype=dtype, device=DEV)
    lse = torch.full((n + 5, hq), 9.0, device=DEV)
    got = b.wrapper.forward(wide[:, 1], b.pages, sm_scale=0.3, out=out[:, 0], lse=lse)
    assert got.data_ptr() == out.data_ptr()
    b.check(out[:, 0], lse, scale=0.3)
    assert (out[n:] == 3).all() and (out[:, 1] == 3).all() and (lse[n:] == 9).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_chunk_attention_hidden_values_do_not_reach_earlier_rows(dtype, bad):
    """K and V of a drafted token that earlier rows do not see may hold anything."""
    b = Batch(8, [70, 300], [4, 6], 8, 2, 128, 16, dtype).begin()
    clean = b.wrapper.forward(b.q, b.pages)
    for i, n in enumerate(b.lens):  # the last token of every request: only its own row sees it
        page = int(b.ids[b.kvp[i] + (n - 1) // 16])
        b.pages[page, :, (n - 1) % 16] = bad
    got = b.wrapper.forward(b.q, b.pages)
    last = (b.qo_dev[1:] - 1).long()
    keep = torch.ones(len(b.q), dtype=torch.bool, device=DEV)
    keep[last] = False
    assert torch.equal(got[keep], clean[keep])
    assert not torch.isfinite(got[last]).any()


def test_chunk_attention_matches_prefill_and_decode():
    """Three kernels, one definition: a mixed batch through prefill, single tokens through decode."""
    b = Batch(9, [512, 90, 1300], [64, 5, 16], 32, 8, 128, 16, torch.bfloat16).begin()
    out = b.wrapper.forward(b.q, b.pages)
    pre = ops.BatchPrefillWithPagedKVCacheWrapper(torch.empty(8 << 20, dtype=torch.uint8, device=DEV))
    pre.begin_forward(b.qo_dev, b.kvp_dev, b.ids, b.last, 32, 8, 128, 16, torch.bfloat16)
    assert (out.float() - pre.forward(b.q, b.pages).float()).abs().max() <= 2e-2
    one = Batch(10, [700, 90, 33], [1, 1, 1], 32, 8, 128, 16, torch.bfloat16).begin()
    dec = ops.BatchDecodeWithPagedKVCacheWrapper(torch.empty(8 << 20, dtype=torch.uint8, device=DEV))
    dec.begin_forward(one.kvp_dev, one.ids, one.last, 32, 8, 128, 16, data_type=torch.bfloat16)
    assert (one.wrapper.forward(one.q, one.pages).float() - dec.forward(one.q, one.pages).float()).abs().max() <= 2e-2


def test_chunk_attention_refuses_a_plan_that_its_tensors_do_not_cover():
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    ws = torch.zeros(4 << 20, dtype=torch.uint8, device=DEV)
    w = dk.BatchChunkWithPagedKVCacheWrapper(ws)
    with pytest.raises(ValueError, match="kv_indices"):
        w.begin_forward(i32([0, 2]), i32([0, 3]), i32([0, 1]), i32([4]), 8, 2, 64, 16, torch.bfloat16)
    with pytest.raises(ValueError, match="batch"):
        w.begin_forward(i32([0, 2]), i32([0, 3]), i32([0, 1, 2]), i32([4, 4]), 8, 2, 64, 16, torch.bfloat16)
    assert not ws.any()  # a refused batch leaves the workspace, and the plan in it, alone
    w.begin_forward(i32([0, 2]), i32([0, 3]), i32([0, 1, 2]), i32([4]), 8, 2, 64, 16, torch.bfloat16)
    pages = torch.zeros(3, 2, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="rows"):
        w.forward(torch.zeros(1, 8, 64, dtype=torch.bfloat16, device=DEV), pages)


def test_chunk_attention_on_a_side_stream_and_in_a_graph():
    b = Batch(11, [5000, 40], [5, 2], 32, 8, 128, 16, torch.bfloat16).begin()
    want = b.wrapper.forward(b.q, b.pages)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = b.wrapper.forward(b.q, b.pages)
    side.synchronize()
    assert torch.equal(got, want)
    out, lse = torch.zeros_like(want), torch.zeros(want.shape[:2], device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.wrapper.forward(b.q, b.pages, out=out, lse=lse)
    for seed in (1, 2):
        b.q.copy_(torch.randn(b.q.shape, generator=torch.Generator().manual_seed(seed)).to(b.q.dtype))
        graph.replay()
        torch.cuda.synchronize()
        b.check(out, lse)


# ---- sampling ------------------------------------------------------------------------------------------------------------------
def _logits(seed, rows, vocab, dtype):
    g = torch.Generator().manual_seed(seed)
    x = 1.3 * torch.empty(rows, vocab).exponential_(generator=g) + 0.5 * torch.randn(rows, vocab, generator=g)
    return x.to(dtype)


def _f32(v):
    return torch.tensor(v, dtype=torch.float32)


def _check_sample(logits, t, k, u):
    """logits on the CPU; returns the tokens."""
    want, p = oracle.sample(logits, t, k, u)
    dev = logits.to(DEV)
    tokens = dk.sample_top_p(dev, t.to(DEV), k.to(DEV), u.to(DEV))
    assert tokens.dtype == torch.int32 and tokens.cpu().tolist() == want.tolist()
    probs = torch.full(logits.shape, -1.0, device=DEV)
    again = dk.sample_top_p(dev, t.to(DEV), k.to(DEV), u.to(DEV), probs=probs)
    assert torch.equal(again, tokens)
    got = probs.cpu().double().numpy()
    assert ((got > 0) == (p > 2.0**-149)).all() or (np.abs(got - p)[(got > 0) != (p > 2.0**-149)] < 1e-38).all()
    # two roundings to fp32 (the quotient, and the exponent's argument where the kernel takes it in fp32: |log p| 2^-24)
    with np.errstate(divide="ignore"):
        log = np.where(p > 0, np.abs(np.log(np.maximum(p, 1e-300))), 0.0)
    assert (np.abs(got - p) <= p * (8 + 4 * log) * 2.0**-24 + 1e-38).all()
    return tokens.cpu()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(3, 1), (5, 7), (9, 1000), (6, 32003), (3, 128256), (2, 262144)])
def test_sample_top_p(dtype, rows, vocab):
    g = torch.Generator().manual_seed(vocab)
    logits = _logits(vocab + 1, rows, vocab, dtype)
    t = _f32([0.8, 1.0, 0.0, 1.3, 0.25, 2.0, 0.7, -1.0, 5.0][:rows])
    k = _f32([0.9, 1.0, 0.5, 0.95, 0.8, 0.3, 0.999, 0.9, 0.99][:rows])
    _check_sample(logits, t, k, torch.rand(rows, generator=g))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top_p", [0.0, 1e-6, 0.5, 0.9, 0.999999, 1.0, 2.0])
def test_sample_top_p_borders(dtype, top_p):
    """Ties at every rank, the random number at both ends, one heavy token, equal tokens, a narrow band of values."""
    vocab = 5003
    g = torch.Generator().manual_seed(1)
    rows = torch.zeros(8, vocab)
    rows[0] = torch.randint(0, 6, (vocab,), generator=g).float()       # six values, ~800 ties each
    rows[1] = 0.0                                                      # all equal
    rows[2, 17] = 40.0                                                 # one token has everything
    rows[3] = torch.randn(vocab, generator=g) * 30                     # few tokens matter
    rows[4] = 1 + torch.arange(vocab).float() * 2.0**-20               # narrow band
    rows[5] = -torch.arange(vocab).float() * 0.01                      # sorted
    rows[6] = torch.randn(vocab, generator=g) * 1e-30                  # weights all 1, values differ
    rows[7] = torch.randn(vocab, generator=g).abs().neg() * 100        # negative values
    for u in (0.0, 0.37, 1 - 2.0**-24):
        _check_sample(rows.to(dtype), torch.ones(8), torch.full((8,), top_p), torch.full((8,), u))


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_top_p_masked_and_odd_rows(dtype):
    """-inf, NaN, +inf and the type's lowest value; a row without tokens; extreme temperatures."""
    vocab, low = 900, torch.finfo(dtype).min
    x = _logits(4, 9, vocab, dtype)
    x[0, 100:] = -float("inf")
    x[1] = -float("inf")
    x[2, ::3] = float("nan")
    x[3, 5], x[3, 800] = float("inf"), float("inf")
    x[4, 3:] = low
    x[5] = low
    x[6] = -float("inf")
    x[6, 899] = -2.0
    t = _f32([1.0, 1.0, 0.7, 0.7, 1.0, 1.0, 1.0, 1e-30, 1e30])
    for top_p in (0.9, 1.0):
        got = _check_sample(x, t, torch.full((9,), top_p), _f32([0.5, 0.5, 0.5, 0.9, 0.9, 0.9, 0.9, 0.9, 0.9]))
        assert got[1] == 0 and got[3] == 800 and got[6] == 899
    _check_sample(x, torch.zeros(9), torch.ones(9), torch.zeros(9))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,stride", [(1001, 1001), (1001, 1003), (4096, 4100), (33, 37)])
def test_sample_top_p_unaligned_rows(dtype, vocab, stride):
    g = torch.Generator().manual_seed(2)
    flat = torch.full((5 * stride + 3,), 50.0).to(dtype)
    x = flat[3:].as_strided((5, vocab), (stride, 1))
    x.copy_(_logits(6, 5, vocab, dtype))
    t, k, u = torch.full((5,), 0.9), torch.full((5,), 0.9), torch.rand(5, generator=g)
    want, _ = oracle.sample(x, t, k, u)
    dev = flat.to(DEV)[3:].as_strided((5, vocab), (stride, 1))
    probs = torch.full((5, stride), -1.0, device=DEV)
    got = dk.sample_top_p(dev, t.to(DEV), k.to(DEV), u.to(DEV), probs=probs[:, :vocab])
    assert got.cpu().tolist() == want.tolist()
    assert (probs[:, vocab:] == -1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(40, 9001), (299, 4099), (700, 1000), (2601, 513)])
def test_sample_top_p_many_rows(dtype, rows, vocab):
    """From rows that are shared by several blocks to one block a row; every third row is flat, so that its border lies among its
    small weights, every seventh holds a few values only, and some random numbers are as small as they get."""
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, vocab, generator=g) * 3
    x[::3] *= 0.05
    x[::7] = torch.randint(0, 9, x[::7].shape, generator=g) * 0.25
    t, k, u = 0.5 + torch.rand(rows, generator=g), 0.3 + 0.7 * torch.rand(rows, generator=g), torch.rand(rows, generator=g)
    t[5::11] = 0.0
    u[::13] = 2.0**-24
    u[1::13] = 0.0
    u[2::13] = 1 - 2.0**-24
    _check_sample(x.to(dtype), t, k, u)


def test_sample_top_p_parameters_that_are_no_numbers():
    x = _logits(7, 4, 640, torch.float32)
    nan = float("nan")
    t, k, u = _f32([nan, 1.0, 1.0, 1.0]), _f32([0.9, nan, 0.9, 0.9]), _f32([0.5, 0.5, nan, 1.5])
    got = dk.sample_top_p(x.to(DEV), t.to(DEV), k.to(DEV), u.to(DEV)).cpu().tolist()
    want, p = oracle.sample(x, t, k, _f32([0.5, 0.5, 0.0, 0.5]))
    assert got[:3] == want[:3].tolist()          # greedy; every token kept; u as 0
    assert got[3] == int(np.nonzero(p[3])[0][-1])  # u at or above 1: the last kept token


# ---- verification --------------------------------------------------------------------------------------------------------------
def _verify_case(seed, drafts, vocab, dtype, with_probs, temps, tops, pad=0):
    g = torch.Generator().manual_seed(seed)
    rows = [n + 1 if n >= 0 else 0 for n in drafts]  # -1: a request without rows
    indptr = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    nnz = int(indptr[-1]) + pad
    logits = _logits(seed, nnz, vocab, dtype)
    owner = np.repeat(np.arange(len(rows)), rows)
    t = torch.tensor([temps[i % len(temps)] for i in range(len(rows))], dtype=torch.float32)
    k = torch.tensor([tops[i % len(tops)] for i in range(len(rows))], dtype=torch.float32)
    z = logits.float() + 0.5 * torch.randn(nnz, vocab, generator=g)
    q = torch.softmax(z, dim=1)
    drafted = torch.multinomial(q, 1, generator=g).squeeze(1)
    for r, o in enumerate(owner):
        if t[o] <= 0 and torch.rand((), generator=g) < 0.7:
            drafted[r] = logits[r].float().argmax()  # greedy drafts that hold
    tokens = torch.cat([drafted[-1:], drafted[:-1]]).to(torch.int32)
    return logits, tokens, indptr, torch.rand(nnz, generator=g), t, k, q if with_probs else None


def _run_verify(logits, tokens, indptr, u, t, k, q):
    dev = [x.to(DEV) if x is not None else None for x in (logits, tokens, torch.from_numpy(indptr), u, t, k)]
    return dk.verify_draft(*dev, draft_probs=None if q is None else q.to(DEV))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_probs", [True, False])
@pytest.mark.parametrize("vocab", [1, 11, 1000, 32003])
def test_verify_draft(dtype, with_probs, vocab):
    drafts = [0, 1, 4, -1, 8, 3, 2, 0, 5, -1, 7, 1]
    case = _verify_case(vocab, drafts, vocab, dtype, with_probs, [1.0, 0.0, 0.7], [1.0, 0.9, 0.95, 0.5], pad=3)
    want_n, want_t = oracle.verify(*case)
    n, tok = _run_verify(*case)
    assert n.dtype == tok.dtype == torch.int32
    assert n.cpu().tolist() == want_n.tolist() and tok.cpu().tolist() == want_t.tolist()


def test_verify_draft_large_vocabulary():
    case = _verify_case(3, [4, 7, 0, 2], 128256, torch.bfloat16, True, [0.8, 1.0], [0.95, 1.0])
    want_n, want_t = oracle.verify(*case)
    n, tok = _run_verify(*case)
    assert n.cpu().tolist() == want_n.tolist() and tok.cpu().tolist() == want_t.tolist()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_probs", [True, False])
def test_verify_draft_many_requests(dtype, with_probs):
    g = torch.Generator().manual_seed(17)
    drafts = (torch.randint(0, 9, (400,), generator=g) - 1).tolist()
    case = _verify_case(18, drafts, 517, dtype, with_probs, [1.0, 0.3, 0.0, 2.5], [1.0, 0.9, 0.4])
    want_n, want_t = oracle.verify(*case)
    n, tok = _run_verify(*case)
    assert n.cpu().tolist() == want_n.tolist() and tok.cpu().tolist() == want_t.tolist()


@pytest.mark.parametrize("with_probs", [True, False])
def test_verify_draft_rejects_tokens_outside_the_vocabulary_and_masked_ones(with_probs):
    logits, tokens, indptr, u, t, k, q = _verify_case(5, [3, 3, 3, 2], 50, torch.float32, with_probs, [1.0], [1.0])
    tokens[1], tokens[5], tokens[6] = -1, 50, 2**31 - 1
    logits[8, int(tokens[9])] = -float("inf")
    logits[13] = -float("inf")  # a row without tokens
    u[:] = 1e-6
    case = (logits, tokens, indptr, u, t, k, q)
    want_n, want_t = oracle.verify(*case)
    n, tok = _run_verify(*case)
    assert n.cpu().tolist() == want_n.tolist() and tok.cpu().tolist() == want_t.tolist()
    assert want_n.tolist()[:3] == [0, 0, 0]


def test_verify_draft_keeps_the_targets_distribution():
    """Whatever the draft proposes, the first emitted token is distributed as the target's nucleus: 200k requests
    with one draft each; a count of n draws is within 5 sigma = 5 sqrt(n p (1 - p)) of n p."""
    vocab, n = 12, 200_000
    g = torch.Generator(device=DEV).manual_seed(3)
    logits = torch.randn(vocab, generator=torch.Generator().manual_seed(1)) * 1.5
    q = torch.softmax(torch.randn(vocab, generator=torch.Generator().manual_seed(2)), 0)
    p = oracle.row_probs(logits, 0.9, 0.9)
    drafts = torch.multinomial(q.to(DEV), n, replacement=True, generator=g).to(torch.int32)
    tokens = torch.stack([torch.zeros_like(drafts), drafts], 1).reshape(-1)
    rows = logits.to(DEV).expand(2 * n, vocab).contiguous()
    acc, nxt = dk.verify_draft(rows, tokens, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=DEV),
                               torch.rand(2 * n, device=DEV, generator=g), torch.full((n,), 0.9, device=DEV),
                               torch.full((n,), 0.9, device=DEV), draft_probs=q.to(DEV).expand(2 * n, vocab).contiguous())
    first = torch.where(acc > 0, drafts, nxt)
    count = torch.bincount(first.long(), minlength=vocab).cpu().numpy()
    assert (np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p)) + 1e-9).all()
    assert 0.2 < float((acc > 0).float().mean()) < 0.95


def test_verify_and_sample_in_a_graph_and_on_a_side_stream():
    case = _verify_case(9, [4, 0, 6], 1000, torch.bfloat16, True, [0.8, 0.0], [0.9])
    logits, tokens, indptr, u, t, k, q = (x.to(DEV) if isinstance(x, torch.Tensor) else torch.from_numpy(x).to(DEV) for x in case)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n, tok = dk.verify_draft(logits, tokens, indptr, u, t, k, q)
    side.synchronize()
    want_n, want_t = oracle.verify(*case)
    assert n.cpu().tolist() == want_n.tolist() and tok.cpu().tolist() == want_t.tolist()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n, tok = dk.verify_draft(logits, tokens, indptr, u, t, k, q)
        drawn = dk.sample_top_p(logits[:3], t, k, u[:3].contiguous())
    for seed in (1, 2):
        u.copy_(torch.rand(len(u), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want_n, want_t = oracle.verify(case[0], case[1], case[2], u.cpu(), *case[4:])
        assert n.cpu().tolist() == want_n.tolist() and tok.cpu().tolist() == want_t.tolist()
        assert drawn.cpu().tolist() == oracle.sample(case[0][:3], case[4], case[5], u[:3].cpu())[0].tolist()
