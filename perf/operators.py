"""Cases of the operators a tree-search decode step needs around the attention: a KV cache held in 4
bits (append, read-back, prefix-aware attention), moving pages of a cache, and the selection of the
next beams.  ``listed()`` and ``draw()`` give the cases, ``prepare()`` what a program holds before the
call, ``run()`` one pass: the plain form, or with ``own`` the package's operators.

The 4-bit cache: one uint8 tensor ``[pages, kv_heads, page_size / 16, 16 * D + 128]`` per layer.  Every
(token, KV head) row of K and of V is stored as 4-bit codes c with its own scale s and offset lo (16-bit
numbers of the model's type): lo = min(x), s = round16((max(x) - lo) / 15), c = rint((x - lo) / s) clipped
to 0..15 (0 where s = 0), value = lo + s * c.  A tile of 16 tokens is [K codes 8D bytes][V codes 8D]
[K (s, lo) pairs 64][V (s, lo) pairs 64].
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a large batch: one new token per request, a few padding slots
        dict(name="append_decode", op="append", tokens=256, heads=8, dim=128, page=16, dtype="bf16", pad=37, run=False),
        # a prefill chunk: long runs of consecutive slots
        dict(name="append_prefill", op="append", tokens=8192, heads=8, dim=128, page=16, dtype="bf16", pad=0, run=True),
        # a short tail read back in front of a chunked prefill; odd length, 64-element heads
        dict(name="gather_tail", op="gather", tokens=777, heads=4, dim=64, page=16, dtype="fp16", pad=5, run=True),
        # a long cached prefix read back as 16-bit rows
        dict(name="gather_prefix", op="gather", tokens=65536, heads=8, dim=128, page=16, dtype="bf16", pad=0, run=True),
        # a small batch with one shared prefix
        dict(name="attn_small", op="attn", tree="1x1024", leaves=8, lo=128, hi=512, median=0, lone=0, lone_lo=1, lone_hi=1,
             q_heads=32, heads=8, dim=128, page=16, dtype="bf16", positions=1),
        # a two-level prefix tree, 64-element heads, speculative steps of three tokens
        dict(name="attn_two_level", op="attn", tree="4x2048,4x512", leaves=8, lo=32, hi=512, median=0, lone=0, lone_lo=1,
             lone_hi=1, q_heads=32, heads=4, dim=64, page=16, dtype="fp16", positions=3),
        # tree search: a complete 4-ary tree with 256 leaves
        dict(name="attn_deep_tree", op="attn", tree="1x256,4x256,4x256,4x256,4x256", leaves=1, lo=64, hi=64, median=0, lone=0,
             lone_lo=1, lone_hi=1, q_heads=64, heads=8, dim=128, page=16, dtype="bf16", positions=1),
        # long contexts: groups with a long shared prefix and log-normal tails, and requests of their own
        dict(name="attn_long", op="attn", tree="7x16384", leaves=32, lo=16, hi=16384, median=2048, lone=32, lone_lo=1024,
             lone_hi=16384, q_heads=64, heads=8, dim=128, page=16, dtype="bf16", positions=1),
        # beams that fork: the last, partly filled page of 61 children, K and V of two layers
        dict(name="copy_fork", op="copy", pairs=61, pool=512, caches=4, kind="bf16", heads=8, dim=128, page=16),
        # compaction of a 16-bit cache: a thousand pages of four tensors move down
        dict(name="copy_compact", op="copy", pairs=1024, pool=2048, caches=4, kind="bf16", heads=8, dim=128, page=16),
        # a small beam search step; odd vocabulary (rows start anywhere), masked tokens
        dict(name="beam_small", op="beam", batch=2, beams=4, vocab=50257, num_out=8, dtype="bf16", masked=0.2, first=False,
             finished=1),
        # a large one: fp32 logits, twice as many candidates as beams
        dict(name="beam_large", op="beam", batch=32, beams=8, vocab=128000, num_out=16, dtype="fp32", masked=0.0, first=False,
             finished=5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "gather", "attn", "attn", "copy", "beam"])
    dtype = rng.choice(["bf16", "fp16"])
    dim = rng.choice([64, 128])
    page = rng.choice([16, 16, 32, 64])
    if op in ("append", "gather"):
        tokens = _log_int(rng, 1, 8192 if op == "append" else 40000)
        return dict(op=op, tokens=tokens, heads=rng.choice([1, 2, 4, 8]), dim=dim, page=page, dtype=dtype,
                    pad=rng.choice([0, 3, 17]), run=rng.random() < 0.5)
    if op == "copy":
        pairs = _log_int(rng, 1, 900)
        return dict(op="copy", pairs=pairs, pool=2 * pairs + rng.randint(0, 100), caches=rng.randint(1, 4),
                    kind=rng.choice(["bf16", "fp16", "int4"]), heads=rng.choice([1, 2, 4, 8]), dim=dim, page=page)
    if op == "beam":
        batch, beams = _log_int(rng, 1, 24), rng.randint(1, 12)
        vocab = _log_int(rng, 1000, 128000)
        if batch * beams * vocab > 20e6:
            batch = max(1, int(20e6 / (beams * vocab)))
        return dict(op="beam", batch=batch, beams=beams, vocab=vocab, num_out=rng.randint(1, 3 * beams),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), masked=rng.choice([0.0, 0.3]), first=rng.random() < 0.2,
                    finished=rng.choice([0, 0, 3]))
    levels = rng.randint(1, 3)
    tree = ",".join("%dx%d" % (rng.randint(1, 4), page * _log_int(rng, 1, max(1, 2048 // page))) for _ in range(levels))
    heads, ratio = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
    return dict(op="attn", tree=tree, leaves=rng.randint(1, 8), lo=1, hi=_log_int(rng, 8, 2000), median=0, lone=rng.randint(0, 8),
                lone_lo=1, lone_hi=_log_int(rng, 8, 6000), q_heads=heads * ratio, heads=heads, dim=dim, page=page, dtype=dtype,
                positions=rng.choice([1, 1, 1, 2, 4]))


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _forest(case, seed):
    """Lengths and page lists of the requests: every root-to-leaf path of the levels in ``tree``
    ("branches x tokens", shared), `leaves` requests below each with a suffix of their own, then
    `lone` requests that share nothing; pages are placed at random."""
    rng = np.random.default_rng(seed)
    page = case["page"]
    count = 0
    paths = [([], 0)]
    for level in case["tree"].split(","):
        branches, tokens = (int(v) for v in level.split("x"))
        n, grown = tokens // page, []
        for pages, length in paths:
            for _ in range(branches):
                grown.append((pages + list(range(count, count + n)), length + tokens))
                count += n
        paths = grown
    lens, tables = [], []

    def add(pages, length, suffix):
        nonlocal count
        n = -(-suffix // page)
        tables.append(pages + list(range(count, count + n)))
        lens.append(length + suffix)
        count += n

    for pages, length in paths:
        for _ in range(case["leaves"]):
            if case["median"]:
                suffix = int(np.clip(round(math.exp(math.log(case["median"]) + 0.8 * rng.standard_normal())), case["lo"], case["hi"]))
            else:
                suffix = int(rng.integers(case["lo"], case["hi"] + 1))
            add(pages, length, suffix)
    for _ in range(case["lone"]):
        add([], 0, int(rng.integers(case["lone_lo"], case["lone_hi"] + 1)))
    place = rng.permutation(count)
    return lens, [place[np.asarray(t, dtype=np.int64)] for t in tables], count


def _unique_tokens(case, lens):
    paths, shared = 1, 0
    for level in case["tree"].split(","):
        branches, tokens = (int(v) for v in level.split("x"))
        paths *= branches
        shared += paths * tokens
    depth = sum(int(level.split("x")[1]) for level in case["tree"].split(","))
    grouped = paths * case["leaves"]
    return shared + sum(n - depth for n in lens[:grouped]) + sum(lens[grouped:])


def _slots(case, seed):
    """Distinct slots of a pool twice as large as needed: single tokens at random places, or runs of
    whole pages in random order; every `pad`-th is a padding slot (-1)."""
    rng = np.random.default_rng(seed)
    tokens, page = case["tokens"], case["page"]
    pages = max(2, -(-2 * tokens // page))
    if case["run"]:
        need = -(-tokens // page)
        base = rng.permutation(pages)[:need].astype(np.int64) * page
        slots = (base[:, None] + np.arange(page)[None, :]).reshape(-1)[:tokens]
    else:
        slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if case["pad"]:
        slots[case["pad"] - 1::case["pad"]] = -1
    return torch.from_numpy(np.ascontiguousarray(slots)).to(DEV), pages


def _empty_cache(pages, case):
    return torch.zeros(pages, case["heads"], case["page"] // 16, 16 * case["dim"] + 128, dtype=torch.uint8, device=DEV)


def _random_cache(pages, case, gen):
    """A filled cache: codes, scales and offsets of N(0, 1) / 2 rows, page by page."""
    cache = _empty_cache(pages, case)
    dtype, page = DTYPES[case["dtype"]], case["page"]
    step = max(1, (1 << 22) // (page * case["heads"] * case["dim"]))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        k, v = (torch.randn(n * page, case["heads"], case["dim"], generator=gen, device=DEV).mul_(0.5).to(dtype) for _ in range(2))
        _write(cache, torch.arange(p * page, (p + n) * page, device=DEV), k, v)
    return cache


def prepare(case, seed):
    state = dict(case)
    gen = _gen(seed)
    op = case["op"]
    if op in ("append", "gather"):
        dtype = DTYPES[case["dtype"]]
        state["slots"], pages = _slots(case, seed)
        shape = (case["tokens"], case["heads"], case["dim"])
        if op == "append":
            state["cache"] = _empty_cache(pages, case)
            state["key"], state["value"] = (torch.randn(shape, generator=gen, device=DEV).mul_(0.5).to(dtype) for _ in range(2))
        else:
            state["cache"] = _random_cache(pages, case, gen)
        # padding rows keep what they held
        state["key_out"], state["value_out"] = (torch.zeros(shape, dtype=dtype, device=DEV) for _ in range(2))
    elif op == "attn":
        lens, tables, pages = _forest(case, seed)
        state["lens"], state["tables"] = lens, [torch.from_numpy(t).to(DEV) for t in tables]
        state["cache"] = _random_cache(pages, case, gen)
        shape = (len(lens), case["positions"], case["q_heads"], case["dim"])
        state["q"] = torch.randn(shape, generator=gen, device=DEV).mul_(0.5).to(DTYPES[case["dtype"]])
        state["scale"] = 1.0 / math.sqrt(case["dim"])
        state["out"] = torch.empty_like(state["q"])
        lse_shape = shape[:3] if case["positions"] > 1 else (shape[0], shape[2])
        state["lse"] = torch.empty(lse_shape, dtype=torch.float32, device=DEV)
        if own:
            from pat_b200 import PrefixTreeCPP
            table = torch.zeros(len(lens), max(len(t) for t in tables), dtype=torch.int32)
            for i, t in enumerate(tables):
                table[i, :len(t)] = torch.from_numpy(t.astype(np.int32))
            tree = PrefixTreeCPP(case["page"])
            tree.build_radix_tree(lens, table)
            tree.pack_schedule(None, case["q_heads"] // case["heads"], case["heads"])
            tree.kernel_info.to_gpu(torch.device(DEV), kv_cache_dtype="int4")
            state["tree"] = tree
    elif op == "copy":
        rng = np.random.default_rng(seed)
        order = rng.permutation(case["pool"])[:2 * case["pairs"]]
        state["mapping"] = torch.from_numpy(order.reshape(-1, 2).astype(np.int64))        # (from, to), planned on the host
        shape, dtype = _page_shape(case)
        make = (lambda: torch.randint(0, 256, (case["pool"], *shape), generator=gen, device=DEV, dtype=torch.uint8)) \
            if dtype is torch.uint8 else \
            (lambda: torch.randn((case["pool"], *shape), generator=gen, device=DEV).to(dtype))
        state["caches"] = [make() for _ in range(case["caches"])]
    else:
        state.update(_beam_inputs(case, gen))
    return state


def _page_shape(case):
    if case["kind"] == "int4":
        return (case["heads"], case["page"] // 16, 16 * case["dim"] + 128), torch.uint8
    return (case["page"], case["heads"], case["dim"]), DTYPES[case["kind"]]


def _beam_inputs(case, gen):
    b, k, v = case["batch"], case["beams"], case["vocab"]
    logits = torch.randn(b, k, v, generator=gen, device=DEV).mul_(2.5)
    if case["masked"]:
        logits.masked_fill_(torch.rand(b, k, v, generator=gen, device=DEV) < case["masked"], float("-inf"))
    scores = torch.randn(b, k, generator=gen, device=DEV).abs_().mul_(-3.0)
    if case["first"]:
        scores[:, 1:] = float("-inf")          # the first step: one live beam per batch entry
    finished = torch.zeros(b, k, dtype=torch.bool, device=DEV)
    if case["finished"]:
        finished.view(-1)[case["finished"] - 1::case["finished"] + 1] = True
    return dict(logits=logits.to(DTYPES[case["dtype"]]), scores=scores, done=finished, pad_token=1)


# ------------------------------------------------------------------------------------- plain forms
def _pack_nibbles(lo, hi):
    return (lo | (hi << 4)).to(torch.uint8)


def _quantise(x):
    """codes (uint8), scale and offset (x's type) of rows along the last dimension."""
    x32 = x.float()
    lo, hi = x32.amin(-1, keepdim=True), x32.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).to(x.dtype)
    s32 = scale.float()
    code = torch.where(s32 > 0, torch.round((x32 - lo) / s32), torch.zeros_like(x32)).clamp(0, 15).to(torch.uint8)
    return code, torch.cat([scale, lo.to(x.dtype)], -1)


def _write(cache, slots, key, value):
    pages, heads, tiles, tile_bytes = cache.shape
    dim = key.shape[-1]
    page, row = slots // (tiles * 16), slots % (tiles * 16)
    tile, tok = row // 16, row % 16
    p, h = page[:, None], torch.arange(heads, device=cache.device)[None, :]
    flat = cache.view(pages, heads, tiles, tile_bytes)
    # K: per 8 dims the bytes (0,2) (4,6) (1,3) (5,7), first of a pair in the low nibble
    code, prm = _quantise(key)
    c = code.view(*code.shape[:2], dim // 8, 2, 2, 2)                          # dim = 8 w + 4 bl + 2 n + hb
    kb = _pack_nibbles(c[..., 0, :], c[..., 1, :]).transpose(-1, -2).reshape(*code.shape[:2], dim // 2)     # [w, hb, bl]
    t = tile[:, None, None]
    off = (tok * (dim // 2))[:, None, None] + torch.arange(dim // 2, device=cache.device)
    flat[p[..., None], h[..., None], t, off] = kb
    off = (16 * dim + tok * 4)[:, None, None] + torch.arange(4, device=cache.device)
    flat[p[..., None], h[..., None], t, off] = prm.contiguous().view(torch.uint8).view(*code.shape[:2], 4)
    # V: 16-bit pieces; token t = 8 half + 2 c + par, dim = (D/8) g + 8 wh + 2 (2 b + n) + wl
    code, prm = _quantise(value)
    c = code.view(*code.shape[:2], 8, dim // 64, 2, 2, 2)                      # g, wh, b, n, wl
    vb = _pack_nibbles(c[..., 0, :], c[..., 1, :])                             # g, wh, b, wl
    vb = vb.transpose(-1, -2).reshape(*code.shape[:2], 8, dim // 32, 2)        # g, w, b
    ar = lambda n: torch.arange(n, device=cache.device)
    half, cc, par = tok // 8, (tok % 8) // 2, tok % 2
    off = (8 * dim + half * 4 * dim + cc * (dim // 8) + par * 2)[:, None, None, None, None] + \
        ar(8)[:, None, None] * (dim // 2) + ar(dim // 32)[:, None] * 4 + ar(2)
    flat[p[..., None, None, None], h[..., None, None, None], tile[:, None, None, None, None], off] = vb
    off = (16 * dim + 64 + tok * 4)[:, None, None] + torch.arange(4, device=cache.device)
    flat[p[..., None], h[..., None], t, off] = prm.contiguous().view(torch.uint8).view(*code.shape[:2], 4)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1)


def _decode(raw, dim, dtype):
    """K and V (fp32) of raw tiles [..., tile_bytes] -> [..., 16, dim]."""
    lead = raw.shape[:-1]
    k = _nibbles(raw[..., :8 * dim]).view(*lead, 16, dim // 8, 2, 2, 2)                   # w, hb, bl, n
    k = k.permute(*range(len(lead)), -5, -4, -2, -1, -3).reshape(*lead, 16, dim).float()
    v = _nibbles(raw[..., 8 * dim:16 * dim]).view(*lead, 2, 8, 4, dim // 64, 2, 2, 2, 2)  # half, g, c, wh, wl, par, b, n
    v = v.permute(*range(len(lead)), -8, -6, -3, -7, -5, -2, -1, -4).reshape(*lead, 16, dim).float()
    prm = raw[..., 16 * dim:].contiguous().view(dtype).view(*lead, 2, 16, 2).float()
    return tuple(prm[..., i, :, 1:] + prm[..., i, :, :1] * x for i, x in enumerate((k, v)))


def _read(cache, slots, dim, dtype):
    tiles = cache.shape[2]
    page, row = slots // (tiles * 16), slots % (tiles * 16)
    keys, values = [], []
    for i in range(0, slots.numel(), 4096):
        k, v = _decode(cache[page[i:i + 4096], :, row[i:i + 4096] // 16], dim, dtype)     # [n, heads, 16, dim]
        at = (row[i:i + 4096] % 16)[:, None, None, None].expand(-1, k.shape[1], 1, dim)
        keys.append(k.gather(2, at)[:, :, 0])
        values.append(v.gather(2, at)[:, :, 0])
    return torch.cat(keys), torch.cat(values)


def _plain_read_back(s):
    keep = s["slots"] >= 0
    k, v = _read(s["cache"], s["slots"][keep], s["dim"], DTYPES[s["dtype"]])
    s["key_out"][keep], s["value_out"][keep] = k.to(s["key_out"].dtype), v.to(s["value_out"].dtype)
    return s["key_out"], s["value_out"]


def _plain_attention(s):
    t_n, dim, page = s["positions"], s["dim"], s["page"]
    group = s["q_heads"] // s["heads"]
    for i, length in enumerate(s["lens"]):
        k, v = _decode(s["cache"][s["tables"][i]], dim, s["q"].dtype)                     # [pages, heads, tiles, 16, dim]
        k, v = (x.permute(1, 0, 2, 3, 4).reshape(s["heads"], -1, dim)[:, :length] for x in (k, v))
        q = s["q"][i].float().view(t_n, s["heads"], group, dim).permute(1, 0, 2, 3).reshape(s["heads"], t_n * group, dim)
        x = torch.matmul(q, k.transpose(1, 2)).mul_(s["scale"]).view(s["heads"], t_n, group, length)
        seen = torch.arange(length, device=x.device)[None, :] < (length - t_n + 1 + torch.arange(t_n, device=x.device))[:, None]
        x = x.masked_fill(~seen[None, :, None, :], float("-inf"))
        top = x.amax(-1, keepdim=True)
        top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
        e = torch.exp(x - top)
        total = e.sum(-1, keepdim=True)
        o = torch.matmul(e.view(s["heads"], t_n * group, length), v).view(s["heads"], t_n, group, dim)
        o = torch.where(total > 0, o / total, torch.zeros_like(o))
        s["out"][i] = o.permute(1, 0, 2, 3).reshape(t_n, s["q_heads"], dim).to(s["out"].dtype)
        lse = (top + torch.log(total))[..., 0].permute(1, 0, 2).reshape(t_n, s["q_heads"])
        s["lse"][i] = lse if t_n > 1 else lse[0]
    return s["out"], s["lse"]


def _plain_copy(s):
    src, dst = s["mapping"].to(DEV).unbind(1)
    for cache in s["caches"]:
        cache[dst] = cache[src]
    return s["caches"]


def _plain_beam(s):
    # in 64 bits: candidates of different beams are compared, and the order has to be right
    b, k, v = s["logits"].shape
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    live = torch.isfinite(top) & torch.isfinite(s["scores"])[..., None]
    logz = top + torch.log(torch.exp(x - torch.where(live, top, torch.zeros_like(top))).sum(-1, keepdim=True))
    value = torch.where(live, s["scores"].double()[..., None] + (x - logz), torch.full_like(x, float("-inf")))
    ended = torch.full_like(x, float("-inf"))
    ended[..., s["pad_token"]] = s["scores"].double()
    value = torch.where(s["done"][..., None], ended, value).view(b, k * v)
    value, order = torch.sort(value, dim=-1, descending=True, stable=True)
    n = s["num_out"]
    order = order[:, :n]
    return value[:, :n].float(), (order // v).int(), (order % v).int()


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "append":
        keep = s["slots"] >= 0
        _write(s["cache"], s["slots"][keep], s["key"][keep], s["value"][keep])
        return _plain_read_back(s)
    if s["op"] == "gather":
        return _plain_read_back(s)
    if s["op"] == "attn":
        return _plain_attention(s)
    if s["op"] == "copy":
        return _plain_copy(s)
    return _plain_beam(s)


def _run_own(s):
    from pat_b200 import beam_select, prefix_attn_with_int4_kvcache
    from pat_b200.cache_ops import copy_pages, gather_cache_int4, reshape_and_cache_int4
    if s["op"] in ("append", "gather"):
        if s["op"] == "append":
            reshape_and_cache_int4(s["key"], s["value"], s["cache"], s["slots"])
        gather_cache_int4(s["cache"], s["slots"], s["key_out"], s["value_out"])
        return s["key_out"], s["value_out"]
    if s["op"] == "attn":
        prefix_attn_with_int4_kvcache(s["q"], s["cache"], s["tree"], s["scale"], s["out"], lse_out=s["lse"])
        return s["out"], s["lse"]
    if s["op"] == "copy":
        copy_pages(s["caches"], s["mapping"])
        return s["caches"]
    return beam_select(s["logits"], s["scores"], s["num_out"], finished=s["done"], pad_token=s["pad_token"])


# ------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op in ("append", "gather"):
        n = case["tokens"] * case["heads"]
        rows, packed = 2 * n * case["dim"] * 2, 2 * n * (case["dim"] // 2 + 4)
        if op == "append":                  # rows in, packed out, and read back: packed in, rows out
            return {"bytes": 2 * rows + 2 * packed + 8 * case["tokens"], "flops": 8 * n * case["dim"]}
        return {"bytes": rows + packed + 8 * case["tokens"], "flops": 4 * n * case["dim"]}
    if op == "attn":
        lens, _, _ = _forest(case, 0)       # (suffix lengths vary a little with the seed)
        packed = 2 * _unique_tokens(case, lens) * case["heads"] * (case["dim"] // 2 + 4)
        rows = len(lens) * case["positions"] * case["q_heads"]
        return {"bytes": packed + rows * (4 * case["dim"] + 4), "flops": 4 * case["dim"] * case["q_heads"] * case["positions"] * sum(lens)}
    if op == "copy":
        shape, dtype = _page_shape(case)
        size = 1 if dtype is torch.uint8 else 2
        return {"bytes": 2 * case["pairs"] * case["caches"] * size * math.prod(shape) + 16 * case["pairs"], "flops": 0}
    n = case["batch"] * case["beams"] * case["vocab"]
    return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + 12 * case["batch"] * case["num_out"], "flops": 3 * n}


# ------------------------------------------------------------------------------- 64-bit definition
def _exact_rows(x):
    """What a row means after 4-bit storage, from the definition (x: 16-bit rows)."""
    y = x.double()
    lo = y.min(-1).values[..., None]
    s = ((y.max(-1).values[..., None] - lo) / 15.0).to(x.dtype).double()
    n = torch.floor((y - lo) / torch.where(s == 0, torch.ones_like(s), s))
    rest = (y - lo) - n * s                         # to the nearest, halves to the even code
    up = (2 * rest > s) | ((2 * rest == s) & (n % 2 == 1))
    return lo + s * (n + up).clamp(max=15)


def _exact_tables(dim):
    """Byte and nibble of element (token, d) of a tile, for K and for V."""
    k = [[(t * (dim // 2) + 4 * (d // 8) + 2 * (d % 2) + (d % 8) // 4, ((d % 8) // 2) % 2) for d in range(dim)] for t in range(16)]
    v = []
    for t in range(16):
        half, c, par = t // 8, (t % 8) // 2, t % 2
        row = []
        for d in range(dim):
            g, r = divmod(d, dim // 8)
            w, j = 2 * (r // 8) + r % 2, (r % 8) // 2
            row.append((8 * dim + half * 4 * dim + (g * 4 + c) * (dim // 8) + 4 * w + 2 * par + j // 2, j % 2))
        v.append(row)
    return [torch.tensor(x, device=DEV) for x in (k, v)]


def _exact_decode(raw, dim, dtype):
    out = []
    for i, table in enumerate(_exact_tables(dim)):
        code = (raw[..., table[..., 0]].int() >> (4 * table[..., 1])) & 15
        at = 16 * dim + 64 * i
        prm = raw[..., at:at + 64].contiguous().view(dtype).double().view(*raw.shape[:-1], 16, 2)
        out.append(code.double() * prm[..., :1] + prm[..., 1:])
    return out


def exact(case, seed):
    if case["op"] == "copy":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        keep = (s["slots"] >= 0)[:, None, None]
        return tuple(torch.where(keep, _exact_rows(s[n]), torch.zeros((), dtype=torch.float64, device=DEV)) for n in ("key", "value"))
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "gather":
        outs = [torch.zeros(s["key_out"].shape, dtype=torch.float64, device=DEV) for _ in range(2)]
        page = case["page"]
        for i in range(0, case["tokens"], 2048):
            slot = s["slots"][i:i + 2048]
            at = slot.clamp(min=0)
            both = _exact_decode(s["cache"][at // page, :, (at % page) // 16], case["dim"], dtype)
            for o, x in zip(outs, both):
                rows = x[torch.arange(slot.numel(), device=DEV), :, at % 16]
                o[i:i + 2048] = torch.where((slot >= 0)[:, None, None], rows, torch.zeros_like(rows))
        return tuple(outs)
    if case["op"] == "attn":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device=DEV)
        group, t_n = case["q_heads"] // case["heads"], case["positions"]
        for i, length in enumerate(s["lens"]):
            for h in range(case["heads"]):
                raw = s["cache"][s["tables"][i], h].reshape(-1, 16 * case["dim"] + 128)
                k, v = (x.reshape(-1, case["dim"])[:length] for x in _exact_decode(raw, case["dim"], dtype))
                for t in range(t_n):
                    n = max(0, length - t_n + 1 + t)
                    heads = slice(h * group, (h + 1) * group)
                    x = s["q"][i, t, heads].double() @ k[:n].T * s["scale"]
                    z = torch.logsumexp(x, -1)
                    out[i, t, heads] = torch.exp(x - z[:, None]) @ v[:n]
                    if t_n > 1:
                        lse[i, t, heads] = z
                    else:
                        lse[i, heads] = z
        return out, lse
    b, k, v = s["logits"].shape
    n = case["num_out"]
    values, parents, tokens = [], [], []
    for i in range(b):
        x = s["logits"][i].double()
        row = s["scores"][i].double()[:, None] + torch.log_softmax(x, -1)
        row = torch.where(torch.isnan(row), torch.full_like(row, float("-inf")), row)
        for j in range(k):
            if bool(s["done"][i, j]):
                row[j] = float("-inf")
                row[j, s["pad_token"]] = s["scores"][i, j].double()
        row = row.view(-1)
        edge = torch.topk(row, n).values[-1]
        if edge == float("-inf"):
            pick = torch.cat([torch.nonzero(row > edge)[:, 0], torch.nonzero(row == edge)[:n, 0]])
        else:
            pick = torch.nonzero(row >= edge)[:, 0]
        val, at = row[pick].cpu().numpy(), pick.cpu().numpy()
        order = np.lexsort((at, -val))[:n]
        values.append(torch.from_numpy(val[order]))
        parents.append(torch.from_numpy((at[order] // v).astype(np.int32)))
        tokens.append(torch.from_numpy((at[order] % v).astype(np.int32)))
    return torch.stack(values).to(DEV), torch.stack(parents).to(DEV), torch.stack(tokens).to(DEV)
