"""Speculative steps through the engine: drafts fed behind the last token, chunk attention over the paged cache,
verification, and the cache positions after a rejection. In fp32 the tokens have to be those of plain greedy decoding."""
import numpy as np
import pytest
import torch

import deserve_b200 as dk
from deserve_b200 import _lib
from oracle import sampling as oracle
from oracle.llama_ref import DenseLlama

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.read_device_status() == 0


def _stages(dtype, cuts, seed=3, sample_seed=None, dim=256, vocab=1000):
    """A 4-layer model cut into stages, a MicroBatchProcessor over a pool of its own for each."""
    args = dk.ModelArgs(dim=dim, n_layers=4, n_heads=4, n_kv_heads=2, vocab_size=vocab, ffn_dim=512, page_size=16)
    procs = []
    for a, b in zip(cuts[:-1], cuts[1:]):
        stage = dk.LlamaStage(args, a, b, DEV, dtype, seed=seed, sample_seed=sample_seed)
        if stage.need_sample:
            stage.output.mul_(12.0)  # decisive logits
        pool = dk.VirtualPagePool(b - a, 64, 0, 16, DEV, dtype, n_kv_heads=2, head_dim=args.head_dim)
        pool.pages.fill_(float("nan"))
        pta = dk.PageTableAllocator(16, 512, 16, DEV)
        mgr = dk.KVCacheManager(pool, dk.CpuChunkPool(b - a, 4, 16, dtype, n_kv_heads=2, head_dim=args.head_dim), pta)
        procs.append(dk.MicroBatchProcessor(mgr, dk.TaskManager(pool.num_pages, 16), stage, pta, True))
    return args, procs


def _plain(procs, prompts, n):
    """Prompt token by token and n greedy tokens, all through the decode path."""
    for p in procs:
        p.join(list(prompts))
        for t, toks in prompts.items():
            p.task_data_manager.add(dk.TaskData.empty(t, len(toks), dk.SamplingParams()))
    out = {t: [] for t in prompts}
    for t, toks in prompts.items():
        feed = list(toks)
        while len(out[t]) < n:
            x = torch.tensor([feed.pop(0)], dtype=torch.int32, device=DEV)
            for p in procs:
                task = p.task_data_manager.get(t)
                task.init(1)
                r = p.exec(x, [t])
                x = r.ongoing_xs if not p.layer_storage.need_sample else r.all_xs
                task.step()
            if not feed:
                tok = int(x[0])
                out[t].append(tok)
                feed.append(tok)
    return out


def _prefill(procs, prompts, params):
    """All but the last prompt token into the cache, so that the first speculative step begins with it."""
    for p in procs:
        p.join(list(prompts))
        for t, toks in prompts.items():
            p.task_data_manager.add(dk.TaskData.empty(t, len(toks) - 1, params(t)))
    for t, toks in prompts.items():
        for tok in toks[:-1]:
            x = torch.tensor([tok], dtype=torch.int32, device=DEV)
            for p in procs:
                task = p.task_data_manager.get(t)
                task.init(1)
                # (a sampling stage may count a token for the last prompt entry: nothing of it is used)
                x = p.exec(x, [t]).ongoing_xs
                task.step()


def _spec_step(procs, ids, fed, **kw):
    """fed: task -> token ids (last token, drafts)."""
    tokens = torch.tensor([x for t in ids for x in fed[t]], dtype=torch.int32, device=DEV)
    x = tokens
    for p in procs:
        for t in ids:
            p.task_data_manager.get(t).init(len(fed[t]))
        r = p.verify(ids, x, tokens=tokens, **kw)
        if not p.layer_storage.need_sample:
            x = r.ongoing_xs
    accepted = r.accepted.tolist()
    done = [p.commit(ids, accepted) for p in procs]
    return r, accepted, done[-1]


@pytest.mark.parametrize("cuts", [(0, 4), (0, 2, 4)])
def test_speculative_greedy_decoding_equals_plain_decoding_fp32(cuts):
    g = torch.Generator().manual_seed(1)
    args, procs = _stages(torch.float32, cuts)
    prompts = {t: torch.randint(1, args.vocab_size, (n,), generator=g).tolist() for t, n in (("a", 5), ("b", 17), ("c", 30))}
    n = 40
    want = _plain(procs, prompts, n)
    for p in procs:
        p.cancel(list(prompts))
        p.task_data_manager.task_datas.clear()
    params = lambda t: dk.SamplingParams(max_new_tokens=n + len(prompts[t]))
    _prefill(procs, prompts, params)
    got, last = {t: [] for t in prompts}, {t: prompts[t][-1] for t in prompts}
    steps = 0
    while any(len(v) < n for v in got.values()):
        ids = [t for t in prompts if len(got[t]) < n]
        fed, right = {}, {}
        for i, t in enumerate(ids):
            k = (steps + 2 * i) % 7                     # drafts: the plain continuation, wrong from some place on
            drafts = want[t][len(got[t]): len(got[t]) + k]
            bad = (steps * 3 + i) % 9
            if bad < len(drafts):
                drafts[bad] = (drafts[bad] + 1) % args.vocab_size
            right[t] = min(bad, len(drafts))
            fed[t] = [last[t]] + drafts
        r, accepted, _ = _spec_step(procs, ids, fed)
        assert isinstance(r, dk.VerifyResult) and r.task_ids == ids and r.logits.shape[0] == sum(map(len, fed.values()))
        for t, a, nxt in zip(ids, accepted, r.tokens.tolist()):
            assert a == right[t], (t, steps)
            got[t] += fed[t][1: 1 + a] + [nxt]
            last[t] = nxt
        steps += 1
    for t in prompts:
        assert got[t][:n] == want[t], t
    assert steps < n  # more than one token per step


def test_speculative_sampling_follows_the_definition():
    """A draft model proposes with its own sampler and probabilities; the target's verdict is the oracle's on its logits. Greedy
    and sampled requests in one step; the tasks end at their token limits."""
    g = torch.Generator().manual_seed(2)
    args, target = _stages(torch.bfloat16, (0, 4), seed=3, sample_seed=5)
    _, draft = _stages(torch.bfloat16, (0, 4), seed=3, sample_seed=6)
    draft[0].layer_storage.layers[3]["w2"].mul_(0.5)  # nearly the same model
    temps, tops = {"a": 0.0, "b": 1.0, "c": 0.7}, {"a": 1.0, "b": 0.9, "c": 1.0}
    prompts = {t: torch.randint(1, args.vocab_size, (n,), generator=g).tolist() for t, n in (("a", 4), ("b", 9), ("c", 20))}
    params = lambda t: dk.SamplingParams(temperature=temps[t], top_p=tops[t], max_new_tokens=1000)
    _prefill(target, prompts, params)
    _prefill(draft, prompts, params)
    ids, last = list(prompts), {t: prompts[t][-1] for t in prompts}
    T = torch.tensor([temps[t] for t in ids])
    P = torch.tensor([tops[t] for t in ids])
    total, dstage = 0, draft[0].layer_storage
    for step in range(6):
        k = 3
        fed, probs = {t: [last[t]] for t in ids}, []
        for _ in range(k):  # the draft model's own steps
            x = torch.tensor([fed[t][-1] for t in ids], dtype=torch.int32, device=DEV)
            for t in ids:
                draft[0].task_data_manager.get(t).init(1)
            batch = draft[0]._batch(ids, x)
            batch.prepare()
            with torch.inference_mode():
                logits = dstage.forward(batch.xs, batch.decode_ctx)
                q = torch.empty(len(ids), args.vocab_size, device=DEV)
                tok = dk.sample_top_p(logits, T.to(DEV), P.to(DEV), dstage.uniform(len(ids), DEV), probs=q)
            batch.decode_ctx.decode_wrapper.end_forward()
            for t, y in zip(ids, tok.tolist()):
                draft[0].task_data_manager.get(t).step()
                fed[t].append(y)
            probs.append(q)
        nnz = len(ids) * (k + 1)
        q = torch.zeros(nnz, args.vocab_size, device=DEV)
        for i in range(len(ids)):
            for j in range(k):
                q[i * (k + 1) + j] = probs[j][i]
        u = torch.rand(nnz, generator=torch.Generator().manual_seed(step)).to(DEV)
        r, accepted, _ = _spec_step(target, ids, fed, draft_probs=q, uniform=u)
        tokens = torch.tensor([y for t in ids for y in fed[t]])
        want_n, want_t = oracle.verify(r.logits, tokens, np.arange(0, nnz + 1, k + 1), u.cpu(), T, P, q)
        assert accepted == want_n.tolist() and r.tokens.tolist() == want_t.tolist()
        total += sum(accepted)
        for i, t in enumerate(ids):
            last[t] = int(r.tokens[i])
            task = draft[0].task_data_manager.get(t)  # the draft's cache goes back to what was accepted
            want_pos = target[0].task_data_manager.get(t).start_pos
            if task.start_pos < want_pos:  # every draft accepted: it has not seen its last one yet
                task.init(1)
                draft[0].exec(torch.tensor([fed[t][-1]], dtype=torch.int32, device=DEV), [t])
                task.step()
            task.start_pos = want_pos
    assert 0 < total < 6 * 3 * 3


def test_sampling_stage_and_greedy_stage():
    """LlamaStage.sample: greedy without a generator, the sampling operator with one (and greedy rows stay greedy)."""
    args, (proc,) = _stages(torch.bfloat16, (0, 4), sample_seed=11)
    _, (plain,) = _stages(torch.bfloat16, (0, 4))
    logits = torch.randn(3, args.vocab_size, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(DEV)
    tasks = [dk.TaskData.empty(str(i), 1, dk.SamplingParams(temperature=t, top_p=0.9)) for i, t in enumerate((0.0, 1.0, 0.5))]
    for t in tasks:
        t.init(1)
    greedy = dk.greedy_sample(logits).tolist()
    assert plain.layer_storage.sample(logits, tasks, True)[0].tolist() == greedy
    state = proc.layer_storage.generator.get_state()
    got = proc.layer_storage.sample(logits, tasks, True)[0].tolist()
    proc.layer_storage.generator.set_state(state)
    u = proc.layer_storage.uniform(3, DEV).cpu()
    want, _ = oracle.sample(logits, torch.tensor([0.0, 1.0, 0.5]), torch.tensor([0.9] * 3), u)
    assert got == want.tolist() and got[0] == greedy[0]


def test_verify_before_the_prompt_is_in_the_cache_is_refused():
    args, (proc,) = _stages(torch.bfloat16, (0, 4))
    proc.join(["a"])
    proc.task_data_manager.add(dk.TaskData.empty("a", 8, dk.SamplingParams()))
    proc.task_data_manager.get("a").init(3)
    with pytest.raises(ValueError, match="behind the whole prompt"):
        proc.verify(["a"], torch.zeros(3, dtype=torch.int32, device=DEV))


def test_commit_ends_tasks_at_their_limits():
    args, (proc,) = _stages(torch.bfloat16, (0, 4))
    for t, limit in (("a", 3), ("b", 100)):
        proc.task_data_manager.add(dk.TaskData.empty(t, 4, dk.SamplingParams(max_new_tokens=limit, max_seq_len=50)))
        proc.task_data_manager.get(t).start_pos = 46
        proc.task_data_manager.get(t).init(4)
    assert proc.commit(["a", "b"], [2, 3]) == ["a", "b"]
    assert [proc.task_data_manager.get(t).start_pos for t in "ab"] == [49, 50]
