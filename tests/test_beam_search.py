"""Beam search over a paged cache: selection of the next beams, the pages they hold, copies of pages, and a
search step put together."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import int4_oracle as I
from pat_b200 import BeamPlanner, PagePool, beam_select
from pat_b200 import _native as N
from pat_b200.cache_ops import _page_geometry, copy_pages, int4_cache_shape, reshape_and_cache_int4

DEV = "cuda:0"
gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------------------- PagePool
def _consistent(pool, tables):
    uses = np.zeros(pool.num_pages, dtype=np.int64)
    for t in tables:
        np.add.at(uses, np.asarray(t, dtype=np.int64), 1)
    assert np.array_equal(uses, pool.uses)


def test_pool_counts_pages():
    pool = PagePool(6, 16)
    a = pool.alloc(2)
    b = pool.alloc(1)
    assert a == [0, 1] and b == [2] and pool.num_free == 3
    pool.share(a)
    pool.free(a)
    assert pool.num_free == 3                           # still held once
    pool.free(a)
    assert pool.num_free == 5 and pool.alloc(3) == [0, 1, 3]
    for bad in (lambda: pool.alloc(3), lambda: pool.free([5]), lambda: pool.free([6]), lambda: pool.share([-1]),
                lambda: pool.free([2, 2])):
        before = pool.uses.copy()
        with pytest.raises(RuntimeError):
            bad()
        assert np.array_equal(before, pool.uses)
    assert pool.alloc(0) == []


def test_extend_takes_a_page_where_the_last_is_full():
    pool = PagePool(4, 4)
    table = []
    slots = [pool.extend(table, n) for n in range(9)]
    assert slots == list(range(9)) and table == [0, 1, 2]


def test_fork_shares_full_pages_and_copies_part_filled_ones():
    pool = PagePool(12, 4)
    tables, lens = [pool.alloc(2), pool.alloc(3), pool.alloc(1)], [6, 12, 1]
    new, new_lens, pairs = pool.fork(tables, lens, [0, 0, 1, 1, 0])
    assert new_lens == [6, 6, 12, 12, 6]
    assert new[0] == tables[0] and new[2] == new[3] == tables[1]       # the first child keeps the page; full ones are shared
    assert [p[0] for p in pairs] == [tables[0][1]] * 2
    assert new[1] == [tables[0][0], pairs[0][1]] and new[4] == [tables[0][0], pairs[1][1]]
    assert not set(p[1] for p in pairs) & set(sum(tables, []))        # targets were free
    _consistent(pool, new)
    assert pool.uses[tables[2][0]] == 0                               # nobody continues request 2


def test_fork_that_does_not_fit_changes_nothing():
    pool = PagePool(3, 4)
    tables, lens = [pool.alloc(2)], [5]
    before = pool.uses.copy()
    with pytest.raises(RuntimeError, match="full"):
        pool.fork(tables, lens, [0, 0, 0])
    assert np.array_equal(before, pool.uses)
    with pytest.raises(RuntimeError, match="parent"):
        pool.fork(tables, lens, [1])


def test_pool_refuses_what_does_not_fit_together():
    pool = PagePool(6, 4)
    tables = [pool.alloc(2)]
    before = pool.uses.copy()
    for bad in [(tables, [9], [0]), (tables, [-1], [0]), (tables, [5, 5], [0]), ([[0, 4]], [5], [0]), ([[0, 7]], [5], [0])]:
        with pytest.raises(RuntimeError):
            pool.fork(*bad)
    with pytest.raises(ValueError):
        pool.alloc(-1)
    assert np.array_equal(before, pool.uses)


@pytest.mark.parametrize("seed", range(5))
def test_random_searches_keep_every_token(seed):
    """A model of the cache on the host: after forks, copies, appends and compactions every request still
    reads its own tokens."""
    rng = np.random.default_rng(seed)
    page, beams = 4, 6
    pool = PagePool(120, page)
    cache = np.full((120, page), -1, dtype=np.int64)
    tables, lens, texts = [[] for _ in range(beams)], [0] * beams, [[] for _ in range(beams)]
    for step in range(40):
        for i in range(beams):
            slot = pool.extend(tables[i], lens[i])
            token = step * beams + i
            cache[slot // page, slot % page] = token
            lens[i] += 1
            texts[i] = texts[i] + [token]
        parents = rng.integers(0, beams, beams).tolist()
        tables, lens, pairs = pool.fork(tables, lens, parents)
        texts = [texts[p] for p in parents]
        for a, b in pairs:
            cache[b] = cache[a]
        if step % 7 == 3:
            tables, pairs = pool.compact(tables)
            for a, b in pairs:
                cache[b] = cache[a]
                cache[a] = -1
            assert pool.num_free == 120 - np.count_nonzero(pool.uses)
            assert not pool.uses[np.count_nonzero(pool.uses):].any()
        _consistent(pool, tables)
        for t, n, text in zip(tables, lens, texts):
            assert cache[t].reshape(-1)[:n].tolist() == text


# -------------------------------------------------------------------------------- refusals, no GPU
def test_page_geometry():
    x = torch.zeros(5, 4, 8, 16, dtype=torch.float16)
    assert _page_geometry(x) == (1, 1024, 1024)
    assert _page_geometry(x[:, :, 2:4]) == (4, 256, 64)              # two heads of every row
    assert _page_geometry(x[:, :, :, :8]) == (32, 32, 16)
    assert _page_geometry(x[:, ::2, 2:4]) == (2, 512, 64)
    assert _page_geometry(x[:, :, ::2, :8]) == (16, 64, 16)
    assert _page_geometry(x[:, :, :3, :8]) is None
    assert _page_geometry(x[:, :1, :1]) == (1, 32, 32)


def test_host_tensors_and_bad_mappings_are_refused(native_lib):
    with pytest.raises(RuntimeError, match="CUDA"):
        copy_pages(torch.zeros(4, 16), [(0, 1)])
    with pytest.raises(RuntimeError, match="pairs"):
        copy_pages(torch.zeros(4, 16), [0, 1, 2])
    with pytest.raises(RuntimeError, match="CUDA"):
        beam_select(torch.zeros(1, 2, 8), torch.zeros(1, 2), 2)
    for bad in ([(0.5, 1.0)], torch.tensor([[0.0, 1.0]]), [(True, False)]):
        with pytest.raises(RuntimeError, match="integers"):
            copy_pages(torch.zeros(4, 16), bad)
    with pytest.raises(TypeError):
        beam_select(torch.zeros(1, 2, 8), torch.zeros(1, 2), 2.5)
    copy_pages([], [(0, 1)])


def _copy_args():
    ptr = (C.c_void_p * 1)(1 << 20)
    pairs = (C.c_int64 * 4)(0, 1, 2, 3)
    a = N.CopyArgs()
    a.caches, a.host_pairs = C.cast(ptr, C.c_void_p), C.cast(pairs, C.c_void_p)
    a.page_stride, a.row_stride, a.row_bytes, a.num_pages = 4096, 4096, 4096, 4
    a.num_caches, a.num_pairs, a.rows = 1, 2, 1
    return a, ptr, pairs


@pytest.mark.parametrize("field,value,code", [
    ("num_pages", 3, -10), ("num_pages", 0, -1), ("rows", 0, -1), ("row_bytes", 0, -1), ("row_bytes", 24, -11),
    ("page_stride", 4088, -11), ("page_stride", 0, -11), ("caches", None, -1), ("host_pairs", None, -1),
    ("device_pairs", 1 << 20, -1), ("num_pairs", -1, -1)])
def test_copy_refuses_bad_arguments(field, value, code, native_lib):
    assert native_lib.pat_b200_copy_pages(None, None) == -1
    a, *keep = _copy_args()
    setattr(a, field, value)
    assert native_lib.pat_b200_copy_pages(C.byref(a), None) == code


def _beam_args(lib):
    a = N.BeamArgs()
    a.logits = a.scores = a.out_scores = a.out_parents = a.out_tokens = a.workspace = 1 << 20
    a.logits_batch_stride, a.logits_beam_stride, a.scores_batch_stride = 400, 100, 4
    a.batch, a.beams, a.vocab, a.num_out, a.dtype, a.pad_token = 2, 4, 100, 8, 2, 0
    a.workspace_bytes = lib.pat_b200_beam_workspace_bytes(2, 4, 100, 8)
    return a


@pytest.mark.parametrize("field,value,code", [
    ("batch", -1, -1), ("beams", 0, -1), ("vocab", 0, -1), ("num_out", 0, -1), ("num_out", 129, -15), ("beams", 513, -15),
    ("vocab", 2 ** 31 - 1, -15), ("logits", None, -1), ("scores", None, -1), ("out_tokens", None, -1), ("pad_token", 100, -1),
    ("pad_token", -1, -1), ("dtype", 3, -11), ("logits", (1 << 20) + 2, -11), ("workspace", None, -12), ("workspace_bytes", 64, -12)])
def test_beam_refuses_bad_arguments(field, value, code, native_lib):
    assert native_lib.pat_b200_beam_select(None, None) == -1
    a = _beam_args(native_lib)
    assert a.workspace_bytes > 0
    setattr(a, field, value)
    assert native_lib.pat_b200_beam_select(C.byref(a), None) == code


def test_beam_asks_for_no_more_than_there_is(native_lib):
    assert native_lib.pat_b200_beam_workspace_bytes(1, 2, 3, 6) > 0
    assert native_lib.pat_b200_beam_workspace_bytes(1, 2, 3, 7) == 0


# ----------------------------------------------------------------------------------------- GPU
@gpu
@pytest.mark.parametrize("shape,dtype", [((9, 16, 8, 128), torch.bfloat16), ((70, 2, 1, 1152), torch.uint8),
                                         ((5, 16, 1, 64), torch.float16), ((600, 64, 4, 64), torch.bfloat16), ((40, 16), torch.uint8)])
@pytest.mark.parametrize("on_device", [False, True])
def test_copies(shape, dtype, on_device, native_lib):
    g = torch.Generator(device=DEV).manual_seed(1)
    caches = [torch.randint(0, 200, shape, generator=g, device=DEV).to(dtype) for _ in range(3)]
    order = np.random.default_rng(2).permutation(shape[0])
    n = shape[0] // 2
    mapping = torch.from_numpy(np.stack([order[:n], order[n:2 * n]], 1).astype(np.int64))
    want = [c.clone() for c in caches]
    for w in want:
        w[mapping[:, 1].to(DEV)] = w[mapping[:, 0].to(DEV)]
    if on_device:
        mapping = torch.cat([mapping, torch.tensor([[-1, 0], [0, shape[0]], [shape[0], 0]])]).to(DEV)
    copy_pages(caches, mapping)
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


@gpu
def test_copies_of_many_caches_and_views(native_lib):
    whole = torch.arange(2 * 6 * 16 * 4 * 64, device=DEV, dtype=torch.float32).view(2, 6, 16, 4, 64).to(torch.bfloat16)
    want = whole.clone()
    want[0, 3, :, 1:3], want[0, 5, :, 1:3] = whole[0, 1, :, 1:3], whole[0, 0, :, 1:3]
    copy_pages(whole[0, :, :, 1:3], [(1, 3), (0, 5)])               # two KV heads of K, V untouched
    assert torch.equal(whole, want)
    many = [torch.full((4, 16, 2, 64), float(i), dtype=torch.float16, device=DEV) for i in range(130)]
    for m in many:
        m[1] += 0.5
    copy_pages(many, torch.tensor([[1, 2]], dtype=torch.int32))
    assert all(torch.equal(m[2], m[1]) and bool((m[3] == float(i)).all()) for i, m in enumerate(many))


@gpu
def test_copy_checks(native_lib):
    c = torch.zeros(8, 16, 2, 64, dtype=torch.float16, device=DEV)
    before = c.clone()
    for bad in ([(0, 8)], [(-1, 2)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(3, 3)], [(0, 1, 2)]):
        with pytest.raises(RuntimeError):
            copy_pages(c, bad)
    for bad in (torch.tensor([[0, 1]], device=DEV, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int64, device=DEV)[::2]):
        with pytest.raises(RuntimeError):
            copy_pages(c, bad)
    with pytest.raises(RuntimeError):
        copy_pages([c, c[:4]], [(0, 1)])
    with pytest.raises(RuntimeError):
        copy_pages(c[:, :, :, 1:9], [(0, 1)])                        # not 16-byte aligned
    copy_pages(c, [])
    copy_pages([c, c.clone()], torch.zeros(0, 2, dtype=torch.int64))
    assert torch.equal(c, before)


def _logits(b, k, v, dtype, seed, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, k, v, generator=g) * 2.5
    if masked:
        x[torch.rand(b, k, v, generator=g) < masked] = float("-inf")
    return x.to(dtype), -torch.rand(b, k, generator=g) * 6


def _check_beam(logits, scores, num_out, finished=None, pad=0, device_logits=None):
    fin = finished.to(DEV) if finished is not None else None
    got = beam_select(logits.to(DEV) if device_logits is None else device_logits, scores.to(DEV), num_out, fin, pad)
    want = I.beam_select(logits, scores, num_out, finished, pad)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int32
    assert torch.equal(got[1].cpu().long(), want[1]) and torch.equal(got[2].cpu().long(), want[2])
    s = got[0].double().cpu()
    seen = want[0] > float("-inf")
    assert torch.equal(s > float("-inf"), seen)
    # one rounding to fp32, of a value that holds an fp32 log-sum accurate to 2^-22
    err = (s - want[0])[seen].abs()
    assert bool((err <= 2.0 ** -24 * want[0][seen].abs() + 2.0 ** -22).all())
    return got


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,k,v,n", [(1, 1, 1, 1), (2, 3, 7, 21), (1, 4, 1000, 8), (3, 2, 8192, 5), (2, 5, 8193, 128), (4, 8, 50257, 16),
                                     (1, 1, 40000, 128), (1, 128, 300, 128)])
def test_selection(b, k, v, n, dtype, native_lib):
    logits, scores = _logits(b, k, v, dtype, v + n)
    _check_beam(logits, scores, n)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_selection_with_masks_and_finished_beams(dtype, native_lib):
    logits, scores = _logits(4, 6, 20001, dtype, 3, masked=0.6)
    logits[0, 1] = float("-inf")                       # a mask that leaves nothing
    logits[1, 2, 777] = float("nan")
    logits[1, 3, 4] = float("inf")
    logits[2, :, 5:] = float("-inf")                   # five tokens a beam
    finished = torch.zeros(4, 6, dtype=torch.bool)
    finished[0, 2] = finished[3, 0] = finished[3, 5] = True
    scores[1, 5] = float("-inf")
    scores[1, 4] = float("nan")
    scores[3, 5] = float("-inf")
    logits[3, 0] = float("nan")                        # a finished beam's logits are not looked at
    _check_beam(logits, scores, 40, finished, 19999)
    _check_beam(logits, scores, 3, finished, 0)


@gpu
def test_first_step_and_empty_entries(native_lib):
    logits, scores = _logits(3, 4, 500, torch.float32, 4)
    scores[:, 1:] = float("-inf")
    _check_beam(logits, scores, 8)
    scores[1] = float("-inf")
    _check_beam(logits, scores, 8)
    logits[2, 0, 3:] = float("-inf")                   # three finite values, eight asked for
    logits[2, 0, 1] = float("-inf")
    _check_beam(logits, scores, 8)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_of_any_finite_size(dtype, native_lib):
    logits, scores = _logits(4, 3, 9000, dtype, 6)
    logits[0, 1, 8500] = 3e38                           # all of its beam's probability
    logits[1, 2] = -3e38                                # its beam's tokens are equal
    logits[2, :, 4:] = -3e38                            # four tokens a beam
    logits[3, 0, 5] = -2.5e38
    logits[3, 1, 7], logits[3, 1, 8] = 1.5e38, -1.5e38
    logits[3, 2] += 1e6
    _check_beam(logits, scores, 16)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_index(dtype, native_lib):
    logits, scores = torch.zeros(2, 3, 20000, dtype=dtype), torch.zeros(2, 3)
    _check_beam(logits, scores, 7)                      # everything is equal
    logits[0, :, 9000:9005] = 3.0
    logits[1, 1, 19999] = logits[1, 1, 0] = 2.0
    _check_beam(logits, scores, 20)
    g = torch.Generator().manual_seed(1)
    row = torch.randn(4097, generator=g).to(dtype)      # equal beams at every alignment: equal sums
    logits = row.expand(2, 6, 4097).contiguous()
    _check_beam(logits, torch.full((2, 6), -1.5), 32)
    steps = (torch.randint(0, 4, (2, 3, 30000), generator=g)).to(dtype)
    _check_beam(steps, torch.zeros(2, 3), 128)


@gpu
def test_selection_of_views(native_lib):
    """The last position of a longer output, a padded vocabulary, transposed beams, strided scores."""
    wide = torch.randn(3, 4, 5, 1024, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    logits = wide[:, :, 2, 3:1004].transpose(0, 1)
    scores = torch.randn(4, 6, generator=torch.Generator().manual_seed(3))[:, ::2]
    dev = wide.to(DEV)[:, :, 2, 3:1004].transpose(0, 1)
    finished = torch.zeros(3, 4, dtype=torch.bool).T
    finished[1, 1] = True
    got = beam_select(dev, scores.to(DEV), 6, finished.to(DEV), 2)
    want = I.beam_select(logits, scores, 6, finished, 2)
    assert torch.equal(got[1].cpu().long(), want[1]) and torch.equal(got[2].cpu().long(), want[2])


@gpu
def test_selection_checks(native_lib):
    x, s = torch.zeros(2, 3, 64, device=DEV), torch.zeros(2, 3, device=DEV)
    for bad in [dict(logits=x[0]), dict(logits=x.double()), dict(scores=s.half()), dict(scores=s[:1]), dict(num_out=0), dict(num_out=193),
                dict(num_out=129), dict(pad_token=64), dict(pad_token=-1), dict(finished=s), dict(finished=torch.zeros(2, 3)),
                dict(logits=x.transpose(1, 2)), dict(logits=x.cpu()), dict(logits=x[:, :0])]:
        with pytest.raises(RuntimeError):
            beam_select(**{**dict(logits=x, scores=s, num_out=4), **bad})
    assert beam_select(x[:0], s[:0], 4)[0].shape == (0, 4)


@gpu
def test_selection_in_a_graph_and_on_two_streams(native_lib):
    logits, scores = _logits(2, 4, 30000, torch.float32, 6)
    xd, sd = logits.to(DEV), scores.to(DEV)
    beam_select(xd, sd, 8)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = beam_select(xd, sd, 8)
        graphs.append((gr, out))
    other, oscores = _logits(2, 4, 30000, torch.float32, 7)
    for x, s in ((other, oscores), (logits, scores)):
        xd.copy_(x)
        sd.copy_(s)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                for _ in range(5):
                    gr.replay()
        torch.cuda.synchronize()
        want = I.beam_select(x, s, 8)
        for _, out in graphs:
            assert torch.equal(out[1].cpu().long(), want[1]) and torch.equal(out[2].cpu().long(), want[2])


@gpu
@pytest.mark.parametrize("kv", ["int4", "auto"])
def test_a_search_end_to_end(kv, native_lib):
    """Beams over one "layer" whose keys and values are functions of the token and its place: after every step
    the attention through the planner's tables equals attention over each beam's own text."""
    from pat_b200 import prefix_attn_with_int4_kvcache, prefix_attn_with_kvcache
    from pat_b200.cache_ops import reshape_and_cache_flash
    batch, beams, vocab, page, hq, hk, d = 2, 4, 61, 16, 8, 2, 64
    g = torch.Generator().manual_seed(0)
    table = [torch.randn(vocab, 256, hk, d, generator=g).mul(0.5).to(torch.float16) for _ in range(2)]     # [token, place]
    pool = PagePool(160, page)
    if kv == "int4":
        caches = [torch.full(int4_cache_shape(160, page, hk, d), 0xFF, dtype=torch.uint8, device=DEV)]
    else:
        caches = [torch.full((160, page, hk, d), float("nan"), dtype=torch.float16, device=DEV) for _ in range(2)]

    def append(tokens, places, slots):
        rows = [t[tokens, places].to(DEV) for t in table]
        if kv == "int4":
            reshape_and_cache_int4(rows[0], rows[1], caches[0], slots.to(DEV))
        else:
            reshape_and_cache_flash(rows[0], rows[1], caches[0], caches[1], slots.to(DEV))

    planner = BeamPlanner(pool, caches, hq // hk, hk, DEV, kv_cache_dtype=kv)
    texts, tables = [], []
    for b in range(batch):
        prompt = torch.randint(0, vocab, (32 + 16 * b,), generator=g)
        pages = pool.alloc(len(prompt) // page)
        append(prompt, torch.arange(len(prompt)), torch.tensor(pages)[:, None].mul(page).add(torch.arange(page)).flatten())
        for k in range(beams):
            if k:
                pool.share(pages)
            texts.append(prompt.tolist())
            tables.append(pages)
    planner.begin(tables, [len(t) for t in texts])
    scores = torch.zeros(batch, beams)
    scores[:, 1:] = float("-inf")
    scores = scores.to(DEV)
    tokens = torch.randint(0, vocab, (batch * beams,), generator=g)
    for step in range(20):
        places = torch.tensor(planner.lens)
        slots = planner.extend()
        append(tokens, places, slots)
        texts = [t + [int(x)] for t, x in zip(texts, tokens)]
        tree = planner.plan()
        q = (torch.randn(batch * beams, 1, hq, d, generator=g) * 0.5).to(torch.float16)
        out = torch.empty(q.shape, dtype=torch.float16, device=DEV)
        if kv == "int4":
            prefix_attn_with_int4_kvcache(q.to(DEV), caches[0], tree, 0.125, out)
        else:
            prefix_attn_with_kvcache(q.to(DEV), caches[0], caches[1], tree, 0.125, out)
        for i, text in enumerate(texts):
            k, v = (t[torch.tensor(text), torch.arange(len(text))] for t in table)
            k, v = ((I.values(x) if kv == "int4" else x.double()) for x in (k, v))
            for h in range(hq):
                w = torch.softmax(k[:, h // 4] @ q[i, 0, h].double() * 0.125, 0)
                err = (out[i, 0, h].double().cpu() - w @ v[:, h // 4]).abs().max()
                assert float(err) <= 4e-3, (step, i, h)           # fp16: u (spread + |out|), spread < 4
        logits = torch.randn(batch, beams, vocab, generator=g) * 2
        old = scores.cpu()
        scores, parents, chosen = planner.select(logits.to(DEV), scores)
        want = I.beam_select(logits, old, beams)
        assert torch.equal(parents.cpu().long(), want[1]) and torch.equal(chosen.cpu().long(), want[2])
        rows = (want[1] + torch.arange(batch)[:, None] * beams).flatten().tolist()
        texts = [texts[r] for r in rows]
        tokens = chosen.cpu().long().flatten()
        _consistent(pool, planner.tables)
