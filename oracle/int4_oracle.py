"""64-bit CPU definition of the 4-bit KV cache and of the beam selection.  TEST INFRASTRUCTURE ONLY: nothing in
the product imports this file.

A (token, KV head) row x of K or of V is held as codes c in 0..15 with lo = min x and
s = round16((max x - lo) / 15), c = the integer nearest to (x - lo) / s, halves to the even one, at most 15;
its values are lo + s c.  The layout of a tile is the one include/pat_b200.h and pat_int4.cuh state.
"""
import numpy as np
import torch


def quantise(x: torch.Tensor):
    """(codes int64, scale float64, offset float64) of 16-bit rows along the last dimension."""
    y = x.double()
    lo = y.amin(-1, keepdim=True)
    s = ((y.amax(-1, keepdim=True) - lo) / 15.0).to(x.dtype).double()
    codes = torch.where(s > 0, torch.round((y - lo) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(y))
    bad = ~torch.isfinite(y).all(-1, keepdim=True)
    nan = torch.full_like(s, float("nan"))
    return (torch.where(bad, torch.zeros_like(codes), codes.clamp(0, 15)).to(torch.int64),
            torch.where(bad, nan, s), torch.where(bad, nan, lo))


def values(x: torch.Tensor) -> torch.Tensor:
    """What rows mean once they are stored (float64)."""
    c, s, lo = quantise(x)
    return lo + s * c.double()


def element_places(dim: int):
    """(byte, nibble) inside a tile of element (token, d): for K, for V.  int64 [16, dim, 2] each."""
    k = np.zeros((16, dim, 2), dtype=np.int64)
    v = np.zeros((16, dim, 2), dtype=np.int64)
    for t in range(16):
        for d in range(dim):
            word, r = divmod(d, 8)
            j, high = divmod(r, 2)                      # nibble j of the low (even d) or high half
            bit = 16 * high + 4 * j
            k[t, d] = (t * dim // 2 + 4 * word + bit // 8, (bit % 8) // 4)
            g, r = divmod(d, dim // 8)
            w, j = 2 * (r // 8) + r % 2, (r % 8) // 2
            bit = 16 * (t % 2) + 4 * j
            lane = 4 * g + (t % 8) // 2
            v[t, d] = (8 * dim + (t // 8) * 4 * dim + lane * dim // 8 + 4 * w + bit // 8, (bit % 8) // 4)
    return k, v


def write(cache: torch.Tensor, slots, key: torch.Tensor, value: torch.Tensor) -> None:
    """In place on a CPU uint8 cache [pages, heads, page / 16, tile]; negative and far slots are skipped."""
    pages, heads, tiles, _ = cache.shape
    dim = key.shape[-1]
    places = element_places(dim)
    flat = cache.numpy()
    for i, slot in enumerate(int(s) for s in slots):
        if slot < 0 or slot >= pages * tiles * 16:
            continue
        page, row = divmod(slot, tiles * 16)
        tile, tok = divmod(row, 16)
        for op, x in enumerate((key, value)):
            codes, s, lo = quantise(x[i])
            prm = torch.cat([s, lo], -1).to(x.dtype).view(torch.uint8).numpy()
            at, nib = places[op][tok, :, 0], places[op][tok, :, 1]
            for h in range(heads):
                raw = flat[page, h, tile]
                for d in range(dim):
                    b = raw[at[d]]
                    c = int(codes[h, d])
                    raw[at[d]] = (b & 0xF0) | c if nib[d] == 0 else (b & 0x0F) | (c << 4)
                off = 16 * dim + 64 * op + 4 * tok
                raw[off:off + 4] = prm[h]


def read(cache: torch.Tensor, dim: int, dtype):
    """K and V (float64) of the whole cache: [pages, page_size, heads, dim] each."""
    pages, heads, tiles, _ = cache.shape
    out = []
    for op, place in enumerate(element_places(dim)):
        place = torch.from_numpy(place)
        codes = (cache[..., place[..., 0]].to(torch.int64) >> (4 * place[..., 1])) & 15
        at = 16 * dim + 64 * op
        prm = cache[..., at:at + 64].contiguous().view(dtype).double().view(pages, heads, tiles, 16, 2)
        x = prm[..., 1:] + prm[..., :1] * codes.double()
        out.append(x.reshape(pages, heads, tiles * 16, dim).permute(0, 2, 1, 3))
    return out


def attention(q, k, v, seq_lens, tables, scale):
    """q [B, T, H, D], k / v [pages, page, Hkv, D] (float64) -> out, lse [B, T, H]; a position that sees
    nothing gives zeros and -inf."""
    B, T, H, D = q.shape
    page, hkv = k.shape[1], k.shape[2]
    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    lse = torch.full((B, T, H), float("-inf"), dtype=torch.float64)
    for b in range(B):
        idx = torch.as_tensor([int(p) for p in tables[b][:-(-seq_lens[b] // page)]], dtype=torch.int64)
        kk, vv = (x[idx].reshape(-1, hkv, D) for x in (k, v))
        for t in range(T):
            n = seq_lens[b] - T + 1 + t
            if n <= 0:
                continue
            for h in range(H):
                s = kk[:n, h // (H // hkv)] @ q[b, t, h].double() * scale
                z = torch.logsumexp(s, 0)
                lse[b, t, h] = z
                out[b, t, h] = torch.exp(s - z) @ vv[:n, h // (H // hkv)]
    return out, lse


def beam_select(logits, scores, num_out, finished=None, pad_token=0):
    """(scores float64, parents, tokens) [batch, num_out], see pat_b200.beam_select."""
    B, K, V = logits.shape
    outs = []
    for b in range(B):
        rows = []
        for k in range(K):
            x, sc = logits[b, k].double(), float(scores[b, k])
            row = torch.full((V,), float("-inf"), dtype=torch.float64)
            if np.isfinite(sc):
                if finished is not None and bool(finished[b, k]):
                    row[pad_token] = sc
                elif not bool((torch.isnan(x) | (x == float("inf"))).any()) and bool((x > float("-inf")).any()):
                    below = x - x.max()             # (first: 64 bits do not hold 3e38 + log n)
                    row = sc + (below - torch.logsumexp(below, 0))
            rows.append(row)
        flat = torch.cat(rows).numpy()
        order = np.lexsort((np.arange(flat.size), -flat))[:num_out]
        outs.append((flat[order], order // V, order % V))
    return tuple(torch.from_numpy(np.stack([o[i] for o in outs])) for i in range(3))
