"""KV cache held in 4 bits: append, read-back and prefix-aware attention, against the 64-bit definition in
oracle/int4_oracle.py."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import int4_oracle as I
from pat_b200 import AsyncTree, DecodePlanner, PrefixTreeCPP, prefix_attn_with_int4_kvcache
from pat_b200 import _native as N
from pat_b200.cache_ops import (gather_cache_int4, int4_cache_shape, int4_tile_bytes, reshape_and_cache_flash,
                                reshape_and_cache_int4)

DEV = "cuda:0"
BF16, FP16 = torch.bfloat16, torch.float16


# ------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("dim", [64, 128])
def test_every_nibble_of_a_tile_belongs_to_one_element(dim, native_lib):
    k, v = I.element_places(dim)
    seen = set()
    for places in (k, v):
        for byte, nibble in places.reshape(-1, 2).tolist():
            assert 0 <= byte < 16 * dim
            seen.add((byte, nibble))
    assert len(seen) == 2 * 16 * dim
    assert int4_tile_bytes(dim) == 16 * dim + 128


def test_cache_shape_and_its_refusals(native_lib):
    assert int4_cache_shape(7, 32, 4, 128) == (7, 4, 2, 2176)
    for page in (0, 8, 24, 272):
        with pytest.raises(RuntimeError):
            int4_cache_shape(7, page, 4, 128)
    with pytest.raises(RuntimeError):
        int4_cache_shape(7, 16, 4, 96)


def test_host_tensors_are_refused(native_lib):
    key = torch.zeros(2, 4, 64, dtype=FP16)
    cache = torch.zeros(int4_cache_shape(2, 16, 4, 64), dtype=torch.uint8)
    slots = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        reshape_and_cache_int4(key, key, cache, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        gather_cache_int4(cache, slots, key, key)
    with pytest.raises(RuntimeError, match="CUDA"):
        prefix_attn_with_int4_kvcache(key[:, None], cache, PrefixTreeCPP(16), 0.1, key[:, None])


def test_unknown_cache_types_are_refused(native_lib):
    tree = PrefixTreeCPP(16)
    tree.build_radix_tree([5], torch.tensor([[0]], dtype=torch.int32))
    tree.pack_schedule(None, 4, 2)
    with pytest.raises(RuntimeError, match="fp8"):
        tree.kernel_info.to_gpu(torch.device("cpu"), kv_cache_dtype="fp8")


def _rows_args():
    a = N.Int4RowsArgs()
    a.key = a.value = a.cache = a.slot_mapping = 1 << 20      # never touched: every call below is refused
    a.key_token_stride = a.value_token_stride = 256
    a.key_head_stride = a.value_head_stride = 64
    a.page_stride, a.head_stride, a.num_pages = 4 * 1152, 1152, 8
    a.num_tokens, a.num_kv_heads, a.head_dim, a.page_size, a.dtype = 3, 4, 64, 16, 0
    return a


@pytest.mark.parametrize("field,value,code", [
    ("num_tokens", -1, -1), ("num_kv_heads", 0, -1), ("num_pages", 0, -1), ("key", None, -1), ("cache", None, -1),
    ("slot_mapping", None, -1), ("head_dim", 96, -11), ("page_size", 8, -11), ("page_size", 272, -11), ("dtype", 2, -11),
    ("key", (1 << 20) + 8, -11), ("key_head_stride", 65, -11), ("value_token_stride", 0, -11), ("head_stride", 1150, -11),
    ("page_stride", -16, -11)])
def test_rows_calls_refuse_bad_arguments(field, value, code, native_lib):
    for fn in (native_lib.pat_b200_append_int4, native_lib.pat_b200_gather_int4):
        assert fn(None, None) == -1
        a = _rows_args()
        setattr(a, field, value)
        assert fn(C.byref(a), None) == code


def test_no_tokens_is_no_work(native_lib):
    a = _rows_args()
    a.num_tokens = 0
    a.key = a.value = a.slot_mapping = None
    assert native_lib.pat_b200_append_int4(C.byref(a), None) == 0


def _decode_args(native_lib):
    tree = PrefixTreeCPP(16)
    tree.build_radix_tree([5, 20], torch.tensor([[0, 0], [1, 2]], dtype=torch.int32))
    tree.pack_schedule(None, 4, 2)
    from pat_b200 import _prefix_attn as P
    work = tree.kernel_info.device_work(torch.device("cpu"), P.int4_config())
    a = N.DecodeInt4Args()
    a.q = a.kv_cache = a.out = a.work_blob = a.workspace = 1 << 20
    a.q_batch_stride = a.out_batch_stride = 512
    a.q_head_stride = a.out_head_stride = 64
    a.page_stride, a.head_stride, a.num_pages = 2 * 1152, 1152, 3
    a.batch, a.q_per_req, a.num_q_heads, a.num_kv_heads, a.head_dim, a.page_size, a.dtype = 2, 1, 8, 2, 64, 16, 0
    a.softmax_scale = 0.125
    a.work = work.header
    a.workspace_bytes = native_lib.pat_b200_workspace_bytes(C.byref(work.header), 8, 64)
    return a


@pytest.mark.parametrize("field,value,code", [
    ("q", None, -1), ("kv_cache", None, -1), ("batch", 0, -1), ("num_q_heads", 7, -1), ("batch", 3, -10), ("q_per_req", 2, -10),
    ("num_kv_heads", 4, -10), ("page_size", 32, -10), ("num_pages", 2, -10), ("head_dim", 80, -11), ("dtype", 2, -11),
    ("softmax_scale", 0.0, -1), ("softmax_scale", float("nan"), -1), ("softmax_scale", float("inf"), -1),
    ("kv_cache", (1 << 20) + 8, -11), ("head_stride", 1160, -11), ("q_head_stride", 60, -11), ("workspace", None, -12),
    ("workspace_bytes", 256, -12)])
def test_attention_refuses_bad_arguments(field, value, code, native_lib):
    assert native_lib.pat_b200_decode_int4(None, None) == -1
    a = _decode_args(native_lib)
    setattr(a, field, value)
    assert native_lib.pat_b200_decode_int4(C.byref(a), None) == code


def test_async_tree_makes_the_plan_of_its_cache(native_lib):
    at = AsyncTree(16, [5, 20], torch.tensor([[0, 0], [1, 2]], dtype=torch.int32), None, 4, 2, torch.device("cpu"), kv_cache_dtype="int4")
    assert isinstance(at.tree, PrefixTreeCPP)
    with pytest.raises(RuntimeError, match="fp8"):
        AsyncTree(16, [5], torch.tensor([[0]], dtype=torch.int32), None, 4, 2, torch.device("cpu"), kv_cache_dtype="fp8").tree


# ------------------------------------------------------------------------------------------ GPU
gpu = pytest.mark.gpu


def _rows(tokens, heads, dim, dtype, seed, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(tokens, heads, dim, generator=g) * spread).to(dtype) for _ in range(2)]


def _fill(pages, page, heads, dim, dtype, seed, byte=0xFF):
    """A CPU cache whose every slot was written, and the GPU copy written by the kernel."""
    key, value = _rows(pages * page, heads, dim, dtype, seed)
    cache = torch.full(int4_cache_shape(pages, page, heads, dim), byte, dtype=torch.uint8, device=DEV)
    reshape_and_cache_int4(key.to(DEV), value.to(DEV), cache, torch.arange(pages * page, device=DEV))
    return cache


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,heads,dim,pages,page,pad", [
    (1, 1, 64, 1, 16, 0), (37, 2, 128, 5, 16, 3), (64, 8, 128, 6, 32, 0), (129, 3, 64, 3, 64, 5), (31, 4, 128, 2, 256, 2)])
def test_append_is_bit_exact(dtype, tokens, heads, dim, pages, page, pad, native_lib):
    key, value = _rows(tokens, heads, dim, dtype, tokens)
    rng = np.random.default_rng(tokens)
    slots = torch.from_numpy(rng.permutation(pages * page)[:tokens].astype(np.int64))
    if pad:
        slots[::pad] = -1
        slots[1::2 * pad] = pages * page + 5           # beyond the cache: skipped as well
    want = torch.full(int4_cache_shape(pages, page, heads, dim), 0xA5, dtype=torch.uint8)
    got = want.to(DEV)
    reshape_and_cache_int4(key.to(DEV), value.to(DEV), got, slots.to(DEV))
    I.write(want, slots.tolist(), key, value)
    assert torch.equal(got.cpu(), want)                 # everything that was not written included


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_append_of_special_rows(dtype, native_lib):
    dim = 128
    g = torch.Generator().manual_seed(1)
    x = torch.randn(12, 1, dim, generator=g)
    x[0] = 0.0
    x[1] = -3.0
    x[2] *= 1e-6                                        # fp16: subnormal rows, the scale rounds to nothing
    x[3] *= 1e4
    x[4, 0, 5] = float("nan")
    x[5, 0, 127] = float("inf")
    x[6, 0, 0] = float("-inf")
    x[7] = torch.linspace(0, 15, dim)                   # halves between two codes
    x[8] = torch.arange(dim) % 2 * 2.0 - 1.0
    x[9, 0, 1:] = 0.0
    x[10] = (torch.arange(dim) % 31).float() / 2.0      # exact halves: scale 1, codes 0, .5, 1, ...
    x[11] = torch.where(torch.arange(dim) == 3, torch.tensor(6e4), torch.tensor(-6e4))
    x = x.to(dtype)
    want = torch.zeros(int4_cache_shape(1, 16, 1, dim), dtype=torch.uint8)
    got = want.to(DEV)
    reshape_and_cache_int4(x.to(DEV), (-x).to(DEV), got, torch.arange(12, device=DEV))
    I.write(want, range(12), x, -x)
    k, v = I.read(got.cpu(), dim, dtype)
    kw, vw = I.read(want, dim, dtype)
    for a, b in ((k, kw), (v, vw)):
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))
    assert torch.isnan(k[0, 4]).all() and torch.isnan(k[0, 5]).all() and torch.isnan(k[0, 6]).all()
    assert not torch.isnan(k[0, :4]).any() and not torch.isnan(k[0, 7:12]).any()
    # the read-back of what was stored
    ko, vo = (torch.zeros(12, 1, dim, dtype=dtype, device=DEV) for _ in range(2))
    gather_cache_int4(got, torch.arange(12, device=DEV), ko, vo)
    assert torch.equal(torch.nan_to_num(ko.cpu()), torch.nan_to_num(kw[0, :12].to(dtype)))
    assert torch.equal(torch.isnan(vo.cpu()), torch.isnan(vw[0, :12]))


@gpu
def test_bf16_rows_over_the_whole_range(native_lib):
    """max - min does not fit in fp32."""
    big = torch.finfo(BF16).max
    x = torch.tensor([-big, big] * 32).view(1, 1, 64).to(BF16)
    cache = torch.zeros(int4_cache_shape(1, 16, 1, 64), dtype=torch.uint8, device=DEV)
    reshape_and_cache_int4(x.to(DEV), x.to(DEV), cache, torch.zeros(1, dtype=torch.int64, device=DEV))
    k, v = I.read(cache.cpu(), 64, BF16)
    assert torch.equal(k[0, 0], I.values(x)[0]) and torch.equal(v[0, 0], I.values(x)[0])


@gpu
def test_rows_with_strides_and_cache_views(native_lib):
    """Keys cut out of a fused projection, a cache with room between pages, one rank's KV heads of a cache."""
    tokens, heads, dim, pages, page = 21, 4, 128, 4, 32
    key, value = _rows(tokens, heads, dim, BF16, 4)
    qkv = torch.zeros(tokens, 3 * heads * dim, dtype=BF16, device=DEV)
    kd, vd = qkv[:, heads * dim:2 * heads * dim].view(tokens, heads, dim), qkv[:, 2 * heads * dim:].view(tokens, heads, dim)
    kd.copy_(key)
    vd.copy_(value)
    shape = int4_cache_shape(pages, page, heads + 2, dim)
    whole = torch.full((2, *shape), 7, dtype=torch.uint8, device=DEV)
    view = whole[1, :, 1:1 + heads]
    slots = torch.from_numpy(np.random.default_rng(0).permutation(pages * page)[:tokens].astype(np.int32)).to(DEV)
    reshape_and_cache_int4(kd, vd, view, slots.view(-1, 1))            # int32 slots, a column of them
    want = torch.full(int4_cache_shape(pages, page, heads, dim), 7, dtype=torch.uint8)
    I.write(want, slots.tolist(), key, value)
    assert torch.equal(view.cpu(), want)
    assert bool((whole[0] == 7).all()) and bool((whole[1, :, 0] == 7).all()) and bool((whole[1, :, 1 + heads:] == 7).all())
    out = torch.full((2, tokens, heads, 2 * dim), 3.0, dtype=BF16, device=DEV)
    gather_cache_int4(view, slots, out[0, ..., :dim], out[1, ..., :dim])
    assert torch.equal(out[0, ..., :dim].cpu(), I.values(key).to(BF16))
    assert torch.equal(out[1, ..., :dim].cpu(), I.values(value).to(BF16))
    assert bool((out[..., dim:] == 3.0).all())


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
def test_gather_leaves_skipped_rows(dtype, dim, native_lib):
    tokens, heads, pages, page = 45, 2, 4, 16
    key, value = _rows(tokens, heads, dim, dtype, 9)
    cache = torch.zeros(int4_cache_shape(pages, page, heads, dim), dtype=torch.uint8, device=DEV)
    slots = torch.arange(3, 3 + tokens)
    reshape_and_cache_int4(key.to(DEV), value.to(DEV), cache, slots.to(DEV))
    ask = slots.clone()
    ask[4], ask[7] = -1, pages * page
    ask[9] = ask[10]                                    # a token may be read twice
    k, v = (torch.full((tokens, heads, dim), 5.0, dtype=dtype, device=DEV) for _ in range(2))
    gather_cache_int4(cache, ask.to(DEV), k, v)
    for got, rows in ((k.cpu(), key), (v.cpu(), value)):
        want = I.values(rows).to(dtype)
        want[9] = want[10]
        want[4] = want[7] = 5.0
        assert torch.equal(got, want)


@gpu
def test_rows_checks(native_lib):
    key, value = (t.to(DEV) for t in _rows(4, 2, 64, FP16, 1))
    cache = torch.zeros(int4_cache_shape(2, 16, 2, 64), dtype=torch.uint8, device=DEV)
    slots = torch.arange(4, device=DEV)
    for bad in [(key, value.bfloat16(), cache, slots), (key.float(), value.float(), cache, slots), (key[0], value[0], cache, slots),
                (key, value[:, :1], cache, slots), (key, value, cache[:, :1], slots), (key, value, cache.float(), slots),
                (key, value, cache[..., :-16], slots), (key, value, cache, slots[:3]),
                (key.transpose(1, 2).contiguous().transpose(1, 2), value, cache, slots)]:
        with pytest.raises(RuntimeError):
            reshape_and_cache_int4(*bad)
    reshape_and_cache_int4(key[:0], value[:0], cache, slots[:0])
    assert int(cache.sum()) == 0
    with pytest.raises(RuntimeError):                   # the 16-bit append does not take the 4-bit cache
        reshape_and_cache_flash(key, value, cache, cache, slots)


# ------------------------------------------------------------------------------------ attention
def _tree(lens, tables, page, ratio, heads, device=DEV):
    table = torch.zeros(len(lens), max(1, max(len(t) for t in tables)), dtype=torch.int32)
    for i, t in enumerate(tables):
        table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
    tree = PrefixTreeCPP(page)
    tree.build_radix_tree(list(lens), table)
    tree.pack_schedule(None, ratio, heads)
    tree.kernel_info.to_gpu(torch.device(device), kv_cache_dtype="int4")
    return tree


def _batch(kind, page, seed):
    """(lens, tables, pages): requests that share whole pages, pages placed at random."""
    rng = np.random.default_rng(seed)
    count, reqs = 0, []

    def take(n):
        nonlocal count
        count += n
        return list(range(count - n, count))

    if kind == "lengths":                               # every end inside a tile and a step, nothing shared
        for n in (1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 600):
            reqs.append((n, take(-(-n // page))))
    elif kind == "pairs":                               # two requests per prefix: up to 16 rows share it
        for n in (16, 48, 160):
            shared = take(-(-n // page))
            for tail in (1, 29):
                reqs.append((len(shared) * page + tail, shared + take(-(-tail // page))))
    elif kind == "shared":                              # one prefix, many requests, a few of them alone
        shared = take(-(-400 // page))
        for tail in (1, 5, 16, 40, 3, 70, 33, 18, 2, 9, 130, 64):
            reqs.append((len(shared) * page + tail, shared + take(-(-tail // page))))
        reqs.append((len(shared) * page, list(shared)))          # ends with the prefix
        reqs.append((77, take(-(-77 // page))))
    else:                                               # a tree of three levels
        for _ in range(2):
            a = take(int(rng.integers(1, 6)))
            for _ in range(3):
                b = a + take(int(rng.integers(1, 4)))
                for _ in range(int(rng.integers(1, 5))):
                    tail = int(rng.integers(1, 90))
                    reqs.append((len(b) * page + tail, b + take(-(-tail // page))))
    place = rng.permutation(count)
    return [n for n, _ in reqs], [[int(place[p]) for p in t] for _, t in reqs], count


def _bounds(k, v, q, scale, dtype, ref):
    """Largest errors of output and LSE.  With u = half a step of the type:

    * P' = p s (or p times s over a power of two) is rounded once (relative u) and multiplies c - 7.5, which moves
      sum p s (c - 7.5) by at most u times half the spread of a value row, itself at most max |v|.  The output is
      rounded once (u |out|).  (2 u max |v| would be p and v = lo + s c rounded once each.)
    * A score is an fp32 sum of 2 D products of at most |q| (16 + 15) s (the codes are exact on both paths):
      2 D roundings of 2^-24 of their sum bound it, and a score's error e changes a weight by a factor of
      1 + 2 e, the output by at most 2 e times the spread of the values.
    * exp2 and the sums over tokens and parts are fp32 as well: 2^-20 of the spread covers them for the lengths used
      here (below 2^10 terms in a random walk, 2^-24 each)."""
    D = q.shape[-1]
    u = torch.finfo(dtype).eps / 2
    spread_v = float((v.amax(-1) - v.amin(-1)).max())
    top_v = float(v.abs().max())
    span_k = float(((v.abs().amax(-1) * 0 + (k.amax(-1) - k.amin(-1)) / 15 * 31) + k.abs().amax(-1)).max())
    e = 2 * D * 2.0 ** -24 * float(q.double().abs().sum(-1).max()) * span_k * scale
    return u * (max(spread_v / 2, 2 * top_v) + ref.abs()) + (2 * e + 2.0 ** -20) * 2 * top_v, e + 2.0 ** -20 * 16


def _check(dtype, hq, hk, d, page, lens, tables, pages, T=1, seed=0, scale=None, cache=None, spread=0.5, q=None):
    g = torch.Generator().manual_seed(seed)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    cache = _fill(pages, page, hk, d, dtype, seed) if cache is None else cache
    if q is None:
        q = (torch.randn(len(lens), T, hq, d, generator=g) * spread).to(dtype)
    tree = _tree(lens, tables, page, hq // hk, hk)
    out = torch.full(q.shape, float("nan"), dtype=dtype, device=DEV)
    lse = torch.full((len(lens), hq) if T == 1 else (len(lens), T, hq), float("nan"), device=DEV)
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    prefix_attn_with_int4_kvcache(q.to(DEV), cache, tree, scale, out, lse_out=lse, _status=status)
    torch.cuda.synchronize()
    assert int(status[0]) == 0
    k, v = I.read(cache.cpu(), d, dtype)
    ref_o, ref_l = I.attention(q, k, v, lens, tables, scale)
    used = torch.tensor(sorted({p for n, t in zip(lens, tables) for p in t[:-(-n // page)]}))
    tol_o, tol_l = _bounds(torch.nan_to_num(k[used]), torch.nan_to_num(v[used]), q, scale, dtype, ref_o)
    err = (out.double().cpu() - ref_o).abs()
    assert bool((err <= tol_o).all()), f"max error {err.max():.3e}, {(err / tol_o).max():.2f} of its bound"
    lse = lse.double().cpu().view(ref_l.shape)
    seen = ref_l > float("-inf")
    assert torch.equal(lse > float("-inf"), seen)
    lerr = (lse - ref_l)[seen].abs()
    assert lerr.numel() == 0 or float(lerr.max()) <= tol_l, f"LSE {float(lerr.max()):.3e} of {tol_l:.3e}"
    return out, lse


CONFIGS = [(BF16, 8, 1, 128, 16), (FP16, 8, 2, 64, 16), (BF16, 4, 4, 64, 32), (FP16, 4, 2, 128, 64), (BF16, 16, 2, 128, 256)]


@gpu
@pytest.mark.parametrize("dtype,hq,hk,d,page", CONFIGS)
@pytest.mark.parametrize("kind", ["lengths", "pairs", "shared", "tree"])
def test_attention(kind, dtype, hq, hk, d, page, native_lib):
    lens, tables, pages = _batch(kind, page, hq + d)
    _check(dtype, hq, hk, d, page, lens, tables, pages, seed=page)


@gpu
@pytest.mark.parametrize("dtype,hq,hk,d,page", CONFIGS)
@pytest.mark.parametrize("T", [2, 3, 7])
def test_several_positions(T, dtype, hq, hk, d, page, native_lib):
    """Positions that see different ends of the context; requests shorter than the step have positions
    that see nothing."""
    lens, tables, pages = _batch("lengths" if T == 3 else "tree" if T == 2 else "shared", page, T)
    _check(dtype, hq, hk, d, page, lens, tables, pages, T=T, seed=T)


@gpu
@pytest.mark.parametrize("dtype,spread,offset", [(FP16, 1e-4, 0.0), (FP16, 200.0, 0.0), (FP16, 0.5, 30.0), (BF16, 1e-20, 0.0),
                                                 (BF16, 1e4, 0.0), (FP16, 0.0, 0.0), (BF16, 0.0, 2.0)])
def test_values_of_any_magnitude(dtype, spread, offset, native_lib):
    """The rounded probabilities carry the values' scales: fp16 has few exponents for them."""
    lens, tables, pages = _batch("shared", 16, 3)
    key, _ = _rows(pages * 16, 2, 128, dtype, 5)
    g = torch.Generator().manual_seed(8)
    value = (torch.randn(pages * 16, 2, 128, generator=g) * spread + offset).to(dtype)
    cache = torch.zeros(int4_cache_shape(pages, 16, 2, 128), dtype=torch.uint8, device=DEV)
    reshape_and_cache_int4(key.to(DEV), value.to(DEV), cache, torch.arange(pages * 16, device=DEV))
    _check(dtype, 8, 2, 128, 16, lens, tables, pages, cache=cache)


@gpu
def test_value_scales_that_grow_along_the_context(native_lib):
    lens, tables = [500], [list(range(32))]
    key, value = _rows(512, 1, 64, FP16, 6)
    value = (value * torch.logspace(-5, 3, 512)[:, None, None]).to(FP16)
    cache = torch.zeros(int4_cache_shape(32, 16, 1, 64), dtype=torch.uint8, device=DEV)
    reshape_and_cache_int4(key.to(DEV), value.to(DEV), cache, torch.arange(512, device=DEV))
    _check(FP16, 4, 1, 64, 16, lens, tables, 32, cache=cache)


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_scores_of_any_size(dtype, native_lib):
    """A softmax that rises all along the context, and one that a single token takes."""
    lens, tables, pages = _batch("lengths", 16, 2)
    key, value = _rows(pages * 16, 2, 64, dtype, 7)
    ramp = torch.zeros(pages * 16)
    for n, t in zip(lens, tables):
        for i, p in enumerate(t):
            ramp[p * 16:(p + 1) * 16] = torch.arange(i * 16, i * 16 + 16) / 10.0
    key[..., 0] = ramp[:, None].to(dtype)
    cache = torch.zeros(int4_cache_shape(pages, 16, 2, 64), dtype=torch.uint8, device=DEV)
    reshape_and_cache_int4(key.to(DEV), value.to(DEV), cache, torch.arange(pages * 16, device=DEV))
    g = torch.Generator().manual_seed(3)
    q = torch.randn(len(lens), 1, 8, 64, generator=g) * 0.2
    q[..., 0] = 4.0
    _check(dtype, 8, 2, 64, 16, lens, tables, pages, cache=cache, q=q.to(dtype))


@gpu
@pytest.mark.parametrize("dim,tokens", [(128, 8192), (64, 5000)])
def test_long_unit_keeps_its_precision(dim, tokens, monkeypatch, native_lib):
    """A unit as long as a whole context, all weights equal: the mean of many values of either sign.

    q = 0 makes every weight 1 and P' = s exactly (the model's type is fp16), so that only fp32 sums and the output's
    rounding are left.  A tensor-core sum of 16 products and its accumulator loses at most 2^-23 of the sum of
    their magnitudes: products up to 79 s, at most 128 tokens' of them before the constant in them is taken out, beside
    the running sum, once a tile.  That is tiles * 2^-23 * (9 * 16 * 79 s + the largest running sum) over the tokens;
    the taking out, twice 2^-24 of as much once in 8 tiles, is within the factor 9 (the sum grows to 8 tiles' only at a
    window's end).  The middles lo + 7.5 s are summed in fp32 per lane: 2^-24 of the largest running sum per token."""
    import pat_b200._prefix_attn as P
    cfg = P.int4_config()
    cfg.num_sms, cfg.items_per_sm, cfg.chunk_tokens_min, cfg.chunk_tokens_max = 1, 1, 1 << 16, 1 << 16
    monkeypatch.setattr(P, "int4_config", lambda: cfg)
    pages = -(-tokens // 16)
    key, value = _rows(pages * 16, 1, dim, FP16, 12)
    cache = torch.zeros(int4_cache_shape(pages, 16, 1, dim), dtype=torch.uint8, device=DEV)
    reshape_and_cache_int4(key.to(DEV), value.to(DEV), cache, torch.arange(pages * 16, device=DEV))
    tree = _tree([tokens], [list(range(pages))], 16, 8, 1)
    q = torch.zeros(1, 1, 8, dim, dtype=FP16, device=DEV)
    out = torch.empty_like(q)
    prefix_attn_with_int4_kvcache(q, cache, tree, 0.1, out)
    v = I.read(cache.cpu(), dim, FP16)[1].reshape(-1, dim)[:tokens].double()
    want = v.mean(0)
    s = float((v.amax(-1) - v.amin(-1)).max() / 15)
    run = float(v.cumsum(0).abs().max() + (v.amax(-1) + v.amin(-1)).cumsum(0).abs().max())
    tol = want.abs() * 2.0 ** -11 + 2.0 ** -23 / 16 * (9 * 16 * 79 * s + run) + 2.0 ** -24 * run
    err = (out[0, 0].double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the bound"


@gpu
@pytest.mark.parametrize("T", [1, 4])
def test_what_lies_behind_a_sequence_is_not_read(T, native_lib):
    """NaN scales behind the last token of every page list (and in pages of nobody) change nothing; with
    several positions a token that only later ones see may be NaN as well."""
    page, hq, hk, d = 16, 8, 2, 128
    lens, tables, pages = _batch("lengths", page, 4)
    lens = [max(n, T) for n in lens]
    cache = _fill(pages, page, hk, d, BF16, 11)
    clean = cache.clone()
    for n, t in zip(lens, tables):
        for slot in range(n, len(t) * page):
            tok = slot % 16
            for off in (16 * d + 4 * tok, 16 * d + 64 + 4 * tok):
                cache[t[slot // page], :, (slot % page) // 16, off:off + 4] = 0xFF
    g = torch.Generator().manual_seed(2)
    q = (torch.randn(len(lens), T, hq, d, generator=g) * 0.5).to(BF16).to(DEV)
    tree = _tree(lens, tables, page, hq // hk, hk)
    outs = []
    for c in (clean, cache):
        out = torch.empty_like(q)
        prefix_attn_with_int4_kvcache(q, c, tree, 0.1, out)
        outs.append(out)
    assert torch.equal(outs[0], outs[1])
    if T > 1:
        last = cache.clone()
        for n, t in zip(lens, tables):
            slot = n - 1
            for off in (16 * d + 4 * (slot % 16), 16 * d + 64 + 4 * (slot % 16)):
                last[t[slot // page], :, (slot % page) // 16, off:off + 4] = 0xFF
        out = torch.empty_like(q)
        prefix_attn_with_int4_kvcache(q, last, tree, 0.1, out)
        assert torch.equal(out[:, :-1], outs[0][:, :-1])
        assert torch.isnan(out[:, -1]).all()


@gpu
def test_nan_that_is_seen_is_returned(native_lib):
    lens, tables = [40, 20], [[0, 1, 2], [3, 4]]
    key, value = _rows(80, 1, 64, BF16, 2)
    key[10] = float("nan")
    cache = torch.zeros(int4_cache_shape(5, 16, 1, 64), dtype=torch.uint8, device=DEV)
    reshape_and_cache_int4(key.to(DEV), value.to(DEV), cache, torch.arange(80, device=DEV))
    q = torch.ones(2, 1, 4, 64, dtype=BF16, device=DEV)
    out = torch.empty_like(q)
    prefix_attn_with_int4_kvcache(q, cache, _tree(lens, tables, 16, 4, 1), 0.1, out)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


@gpu
def test_query_output_and_cache_views(native_lib):
    """Queries inside a fused projection, outputs in a wider buffer, the KV heads of one rank, int4 pages
    with room between them; one head, one request."""
    page, hq, hk, d = 16, 8, 4, 64
    lens, tables, pages = _batch("shared", page, 6)
    whole = torch.full((pages, 2, hk, 1, int4_tile_bytes(d)), 0xFF, dtype=torch.uint8, device=DEV)
    filled = _fill(pages, page, hk, d, FP16, 4)
    whole[:, 1] = filled
    g = torch.Generator().manual_seed(5)
    q = (torch.randn(len(lens), 1, hq, d, generator=g) * 0.5).to(FP16)
    qkv = torch.zeros(len(lens), 1, 3, hq, d, dtype=FP16, device=DEV)
    qkv[:, :, 1] = q.to(DEV)
    buf = torch.full((len(lens), 1, hq, 2 * d), 9.0, dtype=FP16, device=DEV)
    want = torch.empty_like(q, device=DEV)
    prefix_attn_with_int4_kvcache(q.to(DEV), filled, _tree(lens, tables, page, 2, hk), 0.125, want)
    prefix_attn_with_int4_kvcache(qkv[:, :, 1], whole[:, 1], _tree(lens, tables, page, 2, hk), 0.125, buf[..., d:])
    assert torch.equal(buf[..., d:], want) and bool((buf[..., :d] == 9.0).all())
    rank = _tree(lens, tables, page, 2, 2)              # two of four KV heads
    part = torch.empty(len(lens), 1, 4, d, dtype=FP16, device=DEV)
    prefix_attn_with_int4_kvcache(q.to(DEV)[:, :, 4:], whole[:, 1, 2:], rank, 0.125, part)
    assert torch.equal(part, want[:, :, 4:])
    one = _tree(lens[:1], tables[:1], page, 1, 1)
    single = torch.empty(1, 1, 1, d, dtype=FP16, device=DEV)
    prefix_attn_with_int4_kvcache(q.to(DEV)[:1, :, :1], filled[:, :1], one, 0.125, single)
    assert float((single - want[:1, :, :1]).abs().max()) <= 2.0 ** -9


@gpu
def test_streams_graphs_and_growing_batches(native_lib):
    """The planner grows a plan in place; a captured step is replayed after the lengths grew."""
    page, hq, hk, d = 16, 8, 2, 128
    lens, tables, pages = _batch("shared", page, 6)
    tables = [t for n, t in zip(lens, tables) if n % page]
    lens = [n for n in lens if n % page]
    extra = pages
    cache = _fill(pages + 64, page, hk, d, BF16, 4)
    k, v = I.read(cache.cpu(), d, BF16)
    planner = DecodePlanner(page, hq // hk, hk, DEV, kv_cache_dtype="int4")
    g = torch.Generator().manual_seed(5)
    q = (torch.randn(len(lens), 1, hq, d, generator=g) * 0.5).to(BF16)
    qd, out = q.to(DEV), torch.empty(len(lens), 1, hq, d, dtype=BF16, device=DEV)
    graph = None
    for step in range(24):
        for i, n in enumerate(lens):
            if n % page == 0:
                tables[i] = tables[i] + [extra]
                extra += 1
            lens[i] = n + 1
        table = torch.zeros(len(lens), max(len(t) for t in tables), dtype=torch.int32)
        for i, t in enumerate(tables):
            table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        tree = planner.step(lens, table)
        if step == 3:
            prefix_attn_with_int4_kvcache(qd, cache, tree, 0.09, out)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                prefix_attn_with_int4_kvcache(qd, cache, tree, 0.09, out)
        out.fill_(float("nan"))
        if graph is not None and planner.rebuilds == 1:
            graph.replay()
        else:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                prefix_attn_with_int4_kvcache(qd, cache, tree, 0.09, out)
            torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        if step in (0, 4, 11, 23):
            ref, _ = I.attention(q, k, v, lens, tables, 0.09)
            tol, _ = _bounds(torch.nan_to_num(k), torch.nan_to_num(v), q, 0.09, BF16, ref)
            assert bool(((out.double().cpu() - ref).abs() <= tol).all())
    assert planner.advances >= 20


@gpu
@pytest.mark.parametrize("kind", ["lengths", "shared", "tree"])
def test_two_graphs_of_one_plan_replayed_at_once(kind, native_lib):
    """Both were captured on the same stream; each has a workspace of its own."""
    page, hq, hk, d = 16, 16, 2, 128
    lens, tables, pages = _batch(kind, page, 8)
    cache = _fill(pages, page, hk, d, BF16, 4)
    tree = _tree(lens, tables, page, hq // hk, hk)
    g = torch.Generator().manual_seed(5)
    qs = [(torch.randn(len(lens), 1, hq, d, generator=g) * 0.5).to(BF16).to(DEV) for _ in range(2)]
    want, graphs = [], []
    for q in qs:
        out = torch.empty_like(q)
        prefix_attn_with_int4_kvcache(q, cache, tree, 0.09, out)
        want.append(out)
    torch.cuda.synchronize()
    for q in qs:
        out = torch.empty_like(q)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            prefix_attn_with_int4_kvcache(q, cache, tree, 0.09, out)
        graphs.append((gr, out))
    for _ in range(3):
        for _, out in graphs:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(4):
            for (gr, _), st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    gr.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert torch.equal(out, w)


@gpu
def test_append_then_attend(native_lib):
    """A decode step: append the new token of every request, attend over the context that includes it; the
    attention over 4 bits is the 16-bit one over the rows the cache stands for."""
    from pat_b200 import prefix_attn_with_kvcache
    page, hq, hk, d = 16, 16, 4, 128
    lens, tables, pages = _batch("tree", page, 9)
    key, value = _rows(pages * page, hk, d, BF16, 3)
    cache = torch.full(int4_cache_shape(pages, page, hk, d), 0xFF, dtype=torch.uint8, device=DEV)
    last = torch.tensor([t[(n - 1) // page] * page + (n - 1) % page for n, t in zip(lens, tables)])
    old = torch.tensor(sorted(set(range(pages * page)) - set(last.tolist())))
    for part in (old, last):
        reshape_and_cache_int4(key[part].to(DEV), value[part].to(DEV), cache, part.to(DEV))
    g = torch.Generator().manual_seed(5)
    q = (torch.randn(len(lens), 1, hq, d, generator=g) * 0.5).to(BF16)
    out, _ = _check(BF16, hq, hk, d, page, lens, tables, pages, cache=cache, q=q)
    k16, v16 = (torch.empty(pages * page, hk, d, dtype=BF16, device=DEV) for _ in range(2))
    gather_cache_int4(cache, torch.arange(pages * page, device=DEV), k16, v16)
    tree = _tree(lens, tables, page, hq // hk, hk)
    wide = torch.empty_like(out)
    prefix_attn_with_kvcache(q.to(DEV), k16.view(pages, page, hk, d), v16.view(pages, page, hk, d), tree, 1.0 / math.sqrt(d), wide)
    torch.cuda.synchronize()
    # both within 2e-2 of the same exact result; the 16-bit rows are rounded values of the codes
    assert float((out.float() - wide.float()).abs().max()) <= 2e-2


@gpu
def test_attention_with_an_async_tree(native_lib):
    lens, tables, pages = _batch("shared", 16, 4)
    cache = _fill(pages, 16, 2, 64, BF16, 4)
    table = torch.zeros(len(lens), max(len(t) for t in tables), dtype=torch.int32)
    for i, t in enumerate(tables):
        table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
    at = AsyncTree(16, lens, table, None, 4, 2, torch.device(DEV), kv_cache_dtype="int4")
    q = torch.randn(len(lens), 1, 8, 64, dtype=BF16, device=DEV)
    a, b = torch.empty_like(q), torch.empty_like(q)
    prefix_attn_with_int4_kvcache(q, cache, at, 0.125, a)
    prefix_attn_with_int4_kvcache(q, cache, _tree(lens, tables, 16, 4, 2), 0.125, b)
    assert torch.equal(a, b)


@gpu
def test_attention_checks(native_lib):
    page, hq, hk, d = 16, 8, 2, 64
    lens, tables, pages = _batch("pairs", page, 1)
    cache = _fill(pages, page, hk, d, FP16, 2)
    q = torch.zeros(len(lens), 1, hq, d, dtype=FP16, device=DEV)
    out = torch.empty_like(q)
    tree = _tree(lens, tables, page, 4, hk)
    good = dict(q=q, kv_cache=cache, tree=tree, softmax_scale=0.1, out=out)
    prefix_attn_with_int4_kvcache(**good)
    late = PrefixTreeCPP(page)
    late.build_radix_tree(list(lens), [list(t) for t in tables])
    late.pack_schedule(None, 4, hk)
    for bad in [dict(q=q.float()), dict(q=q.cpu()), dict(out=out.bfloat16()), dict(out=out[:1]), dict(kv_cache=cache.cpu()),
                dict(kv_cache=cache.to(torch.int32)), dict(kv_cache=cache[..., :-16]), dict(q=q[..., :32], out=out[..., :32]),
                dict(q=q[:, :, :6], out=out[:, :, :6]), dict(q=q[:2], out=out[:2]), dict(tree=late), dict(tree=None),
                dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(kv_cache=cache[:2]),
                dict(lse_out=torch.empty(len(lens), hq, device=DEV, dtype=FP16)), dict(lse_out=torch.empty(3, device=DEV))]:
        with pytest.raises(RuntimeError):
            prefix_attn_with_int4_kvcache(**{**good, **bad})
