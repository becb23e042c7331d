"""The 4-bit K/V cache's definition in 64 bits (include/foxcuda.h, the 4-bit
cache): the quantiser, the blocks' bytes, and attention over them. Plain numpy
and torch on the CPU; nothing of the library is used."""
import numpy as np

PAGE, GROUP = 64, 64
_F16 = np.sort(np.arange(0x10000, dtype=np.uint32).astype(np.uint16).view(np.float16).astype(np.float64))
_F16 = np.unique(_F16[np.isfinite(_F16)])


def block_bytes(hd):
    return PAGE * (hd // 2 + 4 * (hd // GROUP))


def quantise(x):
    """x [..., hd] (any float type): codes (uint8) [..., hd], d and m (float64) [..., hd / 64]."""
    x = np.clip(np.asarray(x, np.float64), -65504, 65504)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    nan = np.isnan(g).any(-1)
    g = np.where(np.isnan(g), 0.0, g)
    lo, hi = g.min(-1), g.max(-1)
    m = _F16[np.searchsorted(_F16, lo, side="right") - 1]
    # the smallest fp16 d with 15 d >= hi - m (15 d is exact in 64 bits)
    d = _F16[np.searchsorted(15 * _F16, hi - m, side="left")]
    q = (g - m[..., None]) / np.where(d > 0, d, 1)[..., None]
    code = np.where(d[..., None] > 0, np.rint(q), 0)
    assert (code >= 0).all() and (code <= 15).all()
    code = np.where(nan[..., None], 0, code).astype(np.uint8)
    return code.reshape(x.shape), np.where(nan, np.nan, d), np.where(nan, np.nan, m)


def values(code, d, m):
    g = code.reshape(*code.shape[:-1], code.shape[-1] // GROUP, GROUP).astype(np.float64)
    return (m[..., None] + d[..., None] * g).reshape(code.shape)


def code_at(hd, side, p, dim):
    """(byte, high half?) of the code of position p (in its page) and
    dimension dim in a block."""
    slab, r = dim // 128, dim % 128
    wide = min(hd, 128)
    if side == 0:
        word = (r % 64 // 16) * 2 * (wide // 64) + 2 * (r // 64) + r % 16 // 8
        return slab * (PAGE * wide // 2) + p * (wide // 2) + 4 * word + r % 8 // 2, dim % 2
    word = (((slab * 4 + p // 16) * 2 + p // 8 % 2) * 4 + p % 8 // 2) * 8 + r % 32 // 4
    return 4 * (word * (wide // 32) + r // 32) + 2 * (p % 2) + r % 4 // 2, dim % 2


def _places(hd, side):
    p, d = np.meshgrid(np.arange(PAGE), np.arange(hd), indexing="ij")
    return code_at(hd, side, p, d)


def put(cache, table, s, pos, k, v):
    """Quantises k and v [n, kv, hd] into positions pos [n] of sequence s of
    the cache (uint8 [pages, kv, 2, block])."""
    hd = k.shape[-1]
    for side, x in ((0, k), (1, v)):
        code, d, m = quantise(x)
        pair = np.stack([d, m], -1).astype(np.float16).view(np.uint8)  # [n, kv, groups * 4]
        byte, high = _places(hd, side)
        for i, p in enumerate(pos):
            blk = cache[table[s, p // PAGE], :, side]
            b, h = byte[p % PAGE], high[p % PAGE]
            for half in (0, 1):
                keep = 0x0F if half else 0xF0
                at = b[h == half]
                blk[:, at] = (blk[:, at] & keep) | (code[i][:, h == half] << (4 * half))
            n = 4 * (hd // GROUP)
            at = PAGE * hd // 2 + (p % PAGE) * n
            blk[:, at:at + n] = pair[i].reshape(pair.shape[1], -1)


def get(cache, table, s, pos):
    """(k, v) in 64 bits [n, kv, hd] at positions pos of sequence s."""
    hd = cache.shape[3] // 36
    pos = np.asarray(pos)
    blk = cache[table[s, pos // PAGE]]  # [n, kv, 2, bytes]
    out = []
    for side in (0, 1):
        byte, high = _places(hd, side)
        b = np.take_along_axis(blk[:, :, side], np.broadcast_to(byte[pos % PAGE][:, None], blk.shape[:2] + (hd,)), -1)
        code = np.where(high[pos % PAGE][:, None] == 1, b >> 4, b & 15)
        dm = np.ascontiguousarray(blk[:, :, side, PAGE * hd // 2:]).view(np.float16)
        dm = dm.reshape(*blk.shape[:2], PAGE, hd // GROUP, 2)[np.arange(len(pos)), :, pos % PAGE].astype(np.float64)
        out.append(values(code, dm[..., 0], dm[..., 1]))
    return out


def attend(q, cache, table, row_start, kv_len, out, scale=None, seen=None):
    """out [rows, heads, hd] (64 bits) with the rows that belong to sequences
    replaced by their attention. seen(s, positions) -> mask of positions that
    exist (all by default)."""
    import torch
    rows, heads, hd = q.shape
    kv = cache.shape[1]
    scale = scale or 1 / np.sqrt(hd)
    out = out.copy()
    for s in range(len(kv_len)):
        a, b, L = row_start[s], row_start[s + 1], kv_len[s]
        if a == b:
            continue
        if L == 0:
            out[a:b] = 0
            continue
        pos = np.arange(L)
        here = np.ones(L, bool) if seen is None else seen(s, pos)
        k, v = np.zeros((L, kv, hd)), np.zeros((L, kv, hd))
        k[here], v[here] = get(cache, table, s, pos[here])
        k, v = torch.from_numpy(k), torch.from_numpy(v)
        for r in range(a, b):
            last = L - (b - r)
            ok = torch.from_numpy(here & (pos <= last))
            if not ok.any():
                out[r] = 0
                continue
            x = torch.from_numpy(np.asarray(q[r], np.float64)).view(kv, heads // kv, hd)
            z = torch.einsum("hgd,lhd->hgl", x, k[ok]) * scale
            w = torch.softmax(z, -1)
            out[r] = torch.einsum("hgl,lhd->hgd", w, v[ok]).reshape(heads, hd).numpy()
    return out
