"""Paged caches under the models and the decode loops, and the loops' token log probabilities."""

import math

import numpy as np
import pytest
import torch

from oracle import logprobs as olp
from oracle.checks import argmax_violations, rel_err
from skinny_mlx_b200.dense import DenseModel, small_dense
from skinny_mlx_b200.model import SMALL, HybridModel, PagedAttnCache
from skinny_mlx_b200.paged import PagePool, PageTable
from skinny_mlx_b200.spec import (HybridRollback, ScriptedDrafter, ScriptedTreeDrafter, greedy, speculative,
                                  speculative_tree)

PROMPT = [int(x) for x in np.random.default_rng(5).integers(0, SMALL.vocab, 24)]
F8 = torch.float8_e4m3fn


def _pool(model, n_pages=40, page=7, **kw):
    return model.make_pool(n_pages, page, **kw)


@pytest.fixture(scope="module")
def cpu_model():
    return HybridModel(SMALL, seed=0, device="cpu")


def test_pool_and_table_bookkeeping():
    pool = PagePool(2, 5, 2, 64, 4, device="cpu")
    a, b = PageTable(pool, 16), PageTable(pool, 9)
    assert (a.width, b.width, pool.free_pages) == (4, 3, 5)
    a.reserve(5)
    b.reserve(9)
    assert len(a.pages) == 2 and len(b.pages) == 3 and pool.free_pages == 0
    assert sorted(a.pages + b.pages) == list(range(5))
    assert a.device[0].tolist() == a.pages + [-1, -1]
    a.reserve(8)  # (the pages are there)
    with pytest.raises(RuntimeError, match="exhausted"):
        a.reserve(9)
    with pytest.raises(ValueError, match="fit"):
        b.reserve(13)
    b.release()
    a.reserve(16)
    assert len(a.pages) == 4 and pool.free_pages == 1
    for bad in (dict(dtype=torch.float16), dict(head_dim=96), dict(n_pages=0), dict(k_scale=torch.ones(2, 2))):
        with pytest.raises(ValueError):
            PagePool(**{**dict(layers=2, n_pages=5, n_kv_heads=2, head_dim=64, page=4, device="cpu"), **bad})


@pytest.mark.parametrize("shape", [(2,), (3,), (3, 1), (1, 2), (2, 3), (3, 2, 1), (4, 2)])
def test_pool_scales_of_another_shape_are_refused(shape):
    """One scale per layer and kv head: anything else would be spread over dims or layers that it was not made for."""
    for name in ("k_scale", "v_scale"):
        with pytest.raises(ValueError, match=name):
            PagePool(3, 5, 2, 64, 4, dtype=F8, device="cpu", **{name: torch.ones(shape)})
    pool = PagePool(3, 5, 2, 64, 4, dtype=F8, device="cpu", k_scale=torch.full((3, 2), 0.5))
    assert [s.tolist() for s in pool.k_scale] == [[0.5, 0.5]] * 3 and [s.tolist() for s in pool.v_scale] == [[1.0, 1.0]] * 3


def test_caches_refuse_foreign_pools_and_trees(cpu_model):
    with pytest.raises(ValueError, match="pool"):
        cpu_model.make_cache(pool=PagePool(2, 5, 2, 128, 4, device="cpu"))
    with pytest.raises(ValueError, match="pool"):
        DenseModel(small_dense(), seed=3, device="cpu").make_cache(pool=PagePool(2, 5, 2, 128, 4, device="cpu"))
    c = cpu_model.make_cache(pool=_pool(cpu_model))
    cpu_model(torch.tensor(PROMPT), c)
    HybridRollback().record(c)
    with pytest.raises(ValueError, match="contiguous"):
        cpu_model(torch.tensor([1, 2, 3]), c, tree=[-1, 0, 0])


def test_caches_refuse_pools_of_another_device(cpu_model):
    """When the cache is made, not in a step that has already counted its tokens."""
    n = cpu_model.make_pool(4).k.shape[0]
    with pytest.raises(ValueError, match="device"):
        cpu_model.make_cache(pool=PagePool(n, 5, SMALL.n_kv_heads, SMALL.head_dim, 4, device="meta"))
    d = DenseModel(small_dense(), seed=3, device="cpu")
    with pytest.raises(ValueError, match="device"):
        d.make_cache(64, pool=PagePool(2, 5, 8, 128, 16, device="meta"))


def test_cpu_decoding_on_pages_is_the_contiguous_one(cpu_model):
    """The CPU path gathers the pages and computes what the contiguous cache computes: the same bits."""
    m = cpu_model
    ref = greedy(m, PROMPT, 12)
    pool = _pool(m)
    got = greedy(m, PROMPT, 12, cache=m.make_cache(pool=pool))
    assert got == ref
    cache = m.make_cache(pool=pool)
    assert speculative(m, PROMPT, 12, ScriptedDrafter(ref, 0.7, SMALL.vocab, "cpu"), 3, cache=cache) == ref
    used = pool.n_pages - pool.free_pages
    cache.release()
    assert pool.free_pages > pool.n_pages - used and all(c.length == 0 for c in cache.layers if isinstance(c, PagedAttnCache))


def test_a_refused_step_changes_no_state(cpu_model):
    """A step for which the pool has no pages, or a tree, is refused before the recurrent layers have taken it
    in: when pages are there again the sequence goes on as if nothing had happened."""
    m = cpu_model
    x, y = torch.tensor(PROMPT), torch.tensor([5, 6, 7, 8])
    c = m.make_cache()
    m(x, c)
    want = m(y, c)[1]
    pool = m.make_pool(len(PROMPT) // 4 + 1, 4)
    c, other = m.make_cache(pool=pool), m.make_cache(pool=pool)
    m(x, c)  # (fills its pages)
    other.table.reserve(4)
    with pytest.raises(ValueError, match="contiguous"):
        m(y, c, tree=[-1, 0, 1, 2])
    with pytest.raises(RuntimeError, match="exhausted"):
        m(y, c)
    assert c.offset == len(PROMPT)
    other.release()
    assert torch.equal(m(y, c)[1], want)


def test_a_page_is_given_back_once():
    pool = PagePool(1, 6, 2, 64, 4, device="cpu")
    a = pool.take(3)
    for bad in ([a[0], a[0]], [next(i for i in range(6) if i not in a)], [6], [-1], [a[0], 7]):
        with pytest.raises(ValueError, match="given back"):
            pool.give(bad)
        assert pool.free_pages == 3
    pool.give(a[:2])
    with pytest.raises(ValueError, match="given back"):
        pool.give(a)
    pool.give(a[2:])
    assert sorted(pool.take(6)) == list(range(6)) and pool.free_pages == 0
    pool.give([])


def test_a_step_on_released_pages_is_refused(cpu_model):
    """Once a table's pages are back in the pool its cached positions are gone: a step that would read them from
    whatever pages it got next is refused, and goes on when the cache is emptied."""
    m = cpu_model
    pool = m.make_pool(20, 7)
    c = m.make_cache(pool=pool)
    x = torch.tensor(PROMPT)
    want = m(x, c)[1]
    state = [g.state.clone() for g in c.layers if not isinstance(g, PagedAttnCache)]
    c.table.release()
    with pytest.raises(ValueError, match="released"):
        m(torch.tensor([3]), c)
    assert c.offset == len(PROMPT) and pool.free_pages == 20
    assert all(torch.equal(g.state, s) for g, s in zip((g for g in c.layers if not isinstance(g, PagedAttnCache)), state))
    c.reset()
    assert torch.equal(m(x, c)[1], want)
    d = DenseModel(small_dense(), seed=3, device="cpu")
    pool = PagePool(2, 20, 8, 128, 16, device="cpu")
    caches = d.make_cache(64, pool=pool)
    want = d(x, caches)
    caches[0].table.release()
    with pytest.raises(ValueError, match="released"):
        d(torch.tensor([3]), caches)
    for c in caches:
        assert c.length == len(PROMPT)
        c.length = 0
    assert torch.equal(d(x, caches), want)


def test_cpu_loops_report_log_probabilities(cpu_model):
    m = cpu_model
    lps, lps2 = [], []
    ref = greedy(m, PROMPT, 8, logprobs=lps, top_n=3)
    assert speculative(m, PROMPT, 8, ScriptedDrafter(ref, 0.7, SMALL.vocab, "cpu"), 3, logprobs=lps2, top_n=3) == ref
    assert len(lps) == len(lps2) == 8
    cache = m.make_cache()
    _, logits = m(torch.tensor(PROMPT + ref[:-1]), cache)
    lp, ent, top, ids, _ = olp.token_logprobs(logits[len(PROMPT) - 1:].float().numpy(), ref, 3)
    for i, r in enumerate(lps):  # (one token at a time against all at once: bf16 logits a few steps apart)
        assert abs(r.logprob - lp[i]) < 0.2 and abs(r.entropy - ent[i]) < 0.2
        assert r.top[0][0] == ref[i] and math.isclose(r.top[0][1], r.logprob)
        assert [t[1] for t in r.top] == sorted((t[1] for t in r.top), reverse=True)


def _tree_logprobs(model, make_cache, dev):
    """speculative_tree's report against greedy's, for the same tokens.  A verify's logits are within 1.5e-2 of
    the largest logit of a single token's (the verify path's bar), so log probabilities x - lse within twice
    that; the entropy's gradient is -p (ln p + H), of size 2 H at most."""
    lps, lps2, stats = [], [], {}
    ref = greedy(model, PROMPT, 9, cache=make_cache(), logprobs=lps, top_n=3)
    drafter = ScriptedTreeDrafter(ref, 0.6, SMALL.vocab, dev, seed=2)
    assert speculative_tree(model, PROMPT, 9, drafter, 3, stats, cache=make_cache(), logprobs=lps2, top_n=3) == ref
    assert stats["accepted"] > 0 and len(lps) == len(lps2) == 9
    tol = 2 * 1.5e-2 * float(model(torch.tensor(PROMPT + ref[:-1], device=dev), make_cache())[1].float().abs().max())
    for a, b, t in zip(lps, lps2, ref):
        assert abs(a.logprob - b.logprob) <= tol and abs(a.entropy - b.entropy) <= tol * a.entropy and len(b.top) == 3
        assert b.top[0] == (t, b.logprob)


def test_cpu_tree_loop_reports_log_probabilities(cpu_model):
    _tree_logprobs(cpu_model, cpu_model.make_cache, "cpu")


# ---------------------------------------------------------------------------------------------
# on the GPU
# ---------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def gpu_model(cuda_lib):
    from skinny_mlx_b200.patch import patch_model

    m = HybridModel(SMALL, seed=0, device="cuda")
    patch_model(m)
    return m


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 7, 16, 64])
def test_verify_steps_on_pages(gpu_model, dev, page):
    """Prompt, single tokens, 8- and 16-token verify steps with rollbacks: the logits of the paged cache stay
    within the verify path's bar (1.5e-2 of the largest logit, the same argmax but for near-ties) of the
    contiguous one's."""
    m = gpu_model
    caches = [m.make_cache(256), m.make_cache(256, pool=m.make_pool(300 // page + 2, page))]
    rng = np.random.default_rng(page)
    ids = rng.integers(0, SMALL.vocab, 120).tolist()
    at = 0
    for T, keep in ((40, 40), (1, 1), (8, 3), (16, 16), (1, 1), (5, 1), (17, 17), (2, 2)):
        x = torch.tensor(ids[at:at + T], device=dev)
        out = []
        for c in caches:
            rb = HybridRollback()
            rec = 1 < T <= 16
            if rec:
                rb.record(c)
            out.append(m(x, c)[1].float().cpu().numpy())
            if rec:
                rb.rollback(c, fed=T, keep=keep)
        assert rel_err(out[0], out[1]) <= 1.5e-2
        assert not argmax_violations(out[0], out[1])
        at += keep
        assert caches[0].offset == caches[1].offset == at


@pytest.mark.gpu
def test_two_sequences_share_a_pool(gpu_model, dev):
    """Interleaved decoding of two prompts on one pool gives each its own greedy tokens; a released sequence's
    pages serve the next one."""
    m = gpu_model
    pool = m.make_pool(14, 16)
    prompts = [PROMPT, PROMPT[::-1] + PROMPT[:9]]
    want = [greedy(m, p, 10, cache=m.make_cache(pool=pool)) for p in prompts[:1]]
    assert pool.free_pages == 14  # (a dropped cache gives its pages back)
    caches = [m.make_cache(112, pool=pool) for _ in prompts]
    toks, last = [[], []], []
    for p, c in zip(prompts, caches):
        last.append(m(torch.tensor(p, device=dev), c)[1][-1])
    for _ in range(10):
        for i, c in enumerate(caches):
            y = torch.argmax(last[i]).view(1)
            toks[i].append(int(y))
            last[i] = m(y, c)[1][-1]
    assert toks[0] == want[0]
    free = pool.free_pages
    caches[0].release()
    assert pool.free_pages == free + 3  # 34 positions in pages of 16
    again = greedy(m, prompts[1], 10, cache=m.make_cache(112, pool=pool))
    assert again == toks[1]
    for c in caches:
        c.release()
    with pytest.raises(RuntimeError, match="exhausted"):
        m(torch.tensor(PROMPT * 10, device=dev), m.make_cache(pool=pool))


@pytest.mark.gpu
def test_eight_bit_pages(gpu_model, dev):
    """e4m3 pages: the step runs and its logits stay near the bf16 cache's (keys and values carry 2^-4 of
    themselves at most, averaged over the context: a tenth of the largest logit bounds it loosely)."""
    m = gpu_model
    x = torch.tensor(PROMPT, device=dev)
    out = []
    for pool in (m.make_pool(20, 16), m.make_pool(20, 16, dtype=F8), m.make_pool(
            20, 16, dtype=F8, k_scale=torch.full((1, 2), 0.05), v_scale=torch.full((1, 2), 0.02))):
        c = m.make_cache(256, pool=pool)
        m(x, c)
        out.append(m(x[:6], c)[1].float().cpu().numpy())
    assert all(np.isfinite(o).all() and rel_err(out[0], o) < 0.1 for o in out)


@pytest.mark.gpu
def test_fused_steps_refuse_paged_caches(gpu_model, dev):
    from skinny_mlx_b200.fused import FusedStep, GraphedStep

    step = FusedStep(gpu_model)
    c = gpu_model.make_cache(pool=gpu_model.make_pool(20, 16))
    for s in (step, GraphedStep(step)):
        with pytest.raises(ValueError, match="contiguous"):
            s(torch.tensor([1, 2], device=dev), c)


@pytest.mark.gpu
def test_dense_model_on_pages(cuda_lib, dev):
    m = DenseModel(small_dense(), seed=3, device=dev)
    pool = PagePool(2, 20, 8, 128, 16, device=dev)
    caches = [m.make_cache(128), m.make_cache(128, pool=pool)]
    rng = np.random.default_rng(1)
    for T in (30, 1, 8, 16):
        x = torch.tensor(rng.integers(0, 4096, T), device=dev)
        a, b = (m(x, c).float().cpu().numpy() for c in caches)
        assert rel_err(a, b) <= 1.5e-2 and not argmax_violations(a, b)
    assert caches[1][0].length == 55 and pool.free_pages == 16
    caches[1][0].table.release()
    assert pool.free_pages == 20


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
def test_loops_report_log_probabilities(gpu_model, dev, fused):
    """The reported values are the f64 oracle's on the very logits of the step (the model is wrapped to keep
    them), for the tokens that were emitted."""
    from skinny_mlx_b200.fused import FusedStep, GraphedStep

    m = GraphedStep(FusedStep(gpu_model)) if fused else gpu_model

    class Keep:
        def __init__(self):
            self.seen = []

        def __getattr__(self, name):
            return getattr(m, name)

        def __call__(self, ids, cache):
            h, logits = m(ids, cache)
            self.seen.append(logits.float().cpu().numpy())
            return h, logits

    k, lps = Keep(), []
    ref = greedy(k, PROMPT, 9, logprobs=lps, top_n=4)
    rows = np.stack([s[-1] for s in k.seen[:9]])
    _check(lps, rows, ref)
    k, lps, stats = Keep(), [], {}
    got = speculative(k, PROMPT, 9, ScriptedDrafter(ref, 0.6, SMALL.vocab, dev), 3, stats=stats, logprobs=lps, top_n=4)
    assert len(lps) == 9
    # a step's emitted tokens are the argmaxes of its first rows: walk the steps with the drafter's luck
    rows, drafter = [k.seen[0][-1]], ScriptedDrafter(ref, 0.6, SMALL.vocab, "cpu")
    drafter.begin(PROMPT, None, got[0])
    for s in k.seen[1:]:
        draft, n = drafter.draft(3).tolist(), 0
        while n < 3 and draft[n] == int(np.argmax(s[n])):
            n += 1
        rows += list(s[:n + 1])
        drafter.update(None, [0] * (n + 1))
    assert len(rows) >= 9 and [int(np.argmax(r)) for r in rows[:9]] == got
    _check(lps, np.stack(rows[:9]), got)


@pytest.mark.gpu
def test_tree_loop_reports_log_probabilities(gpu_model, dev):
    from skinny_mlx_b200.fused import FusedStep, GraphedStep

    _tree_logprobs(GraphedStep(FusedStep(gpu_model)), gpu_model.make_cache, dev)


def _check(lps, rows, tokens):
    lp, ent, top, ids, spread = olp.token_logprobs(rows, tokens, 4)
    for i, r in enumerate(lps):
        # f32 sums of at most V / 256 + 64 terms in a chain, values rounded four times (as in the operator's test)
        tol = (4096 / 256 + 68 + 2 * spread[i]) * 2.0 ** -24 + 4 * (2 * np.abs(rows[i]).max() + 9) * 2.0 ** -24
        assert abs(r.logprob - lp[i]) <= tol and abs(r.entropy - ent[i]) <= tol * (2 + 4 * spread[i])
        assert [t for t, _ in r.top] == ids[i].tolist()
        assert all(abs(a - b) <= tol for (_, a), b in zip(r.top, top[i]))
