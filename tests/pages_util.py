"""A paged cache and its ragged batches in plain 64-bit arithmetic, for the tests of the paged operators."""
import numpy as np
import torch

BLOCK = 16


def turned(x, pos, theta, neox):
    """x [rows, heads, hd] rotated at pos [rows], in 64 bits"""
    x = x.double()
    if theta == 0:
        return x
    hd, theta = x.shape[-1], float(np.float32(theta))  # the base is an f32 number
    a = pos.double()[:, None] * theta ** (-torch.arange(hd // 2, dtype=torch.float64, device=x.device) * 2 / hd)
    c, s = a.cos()[:, None], a.sin()[:, None]
    u, w = (x[..., :hd // 2], x[..., hd // 2:]) if neox else (x[..., 0::2], x[..., 1::2])
    u, w = u * c - w * s, u * s + w * c
    return torch.cat((u, w), -1) if neox else torch.stack((u, w), -1).flatten(-2)


class Cache:
    """pools on `device` with a shuffled page table for sequences of up to `longest` positions"""

    def __init__(self, n_seq, longest, page, n_kv, hd, dtype, seed=0, spare=2, device="cuda", junk=True):
        from mesh_llm_b200 import ops

        per = (longest + page - 1) // page
        g = np.random.default_rng(seed)
        self.n_pages, self.page, self.n_kv, self.hd, self.dtype = n_seq * per + spare, page, n_kv, hd, dtype
        self.k, self.v, self.ks, self.vs = ops.kv_pages(self.n_pages, page, n_kv, hd, dtype, device)
        if junk:  # what a page held for someone else: NaN everywhere
            for t in (self.k, self.v):
                t.view(torch.uint8 if dtype == torch.float8_e4m3fn else torch.int16).fill_(0x7F if dtype == torch.float8_e4m3fn else 0x7E00)
            for t in (self.ks, self.vs):
                if t is not None:
                    t.fill_(128.0)
        self.table = torch.from_numpy(g.permutation(self.n_pages)[:n_seq * per].reshape(n_seq, per).astype(np.int32)).to(device)

    def values(self):
        """what the pools hold, in 64 bits: two [n_pages, n_kv, page, hd]"""
        out = []
        for t, s in ((self.k, self.ks), (self.v, self.vs)):
            x = t.double()
            out.append(x if s is None else x * s.double().repeat_interleave(BLOCK, -1)[..., None])
        return out

    def rows(self, s, n, values=None):
        """keys and values of the first n positions of sequence s: [n, n_kv, hd]"""
        pos = torch.arange(n, device=self.k.device)
        at = self.table[s].long()[pos // self.page], pos % self.page
        return [x[at[0], :, at[1]] for x in (values or self.values())]

    @property
    def scales(self):
        return dict(k_scale=self.ks, v_scale=self.vs)

    def append(self, k, v, batch, theta, neox):
        from mesh_llm_b200 import ops

        ops.kv_pages_append(k, v, self.k, self.v, self.table, batch.start, batch.pos0, theta, neox, **self.scales)

    def attend(self, q, batch, theta, neox, window=0, max_rows=None, **kw):
        from mesh_llm_b200 import ops

        return ops.attention_pages(q, self.k, self.v, self.table, batch.start, batch.pos0, batch.most if max_rows is None else max_rows, theta, neox,
                                   window=window, **self.scales, **kw)


class Batch:
    def __init__(self, new, past, device="cuda", first=0):
        self.new, self.past, self.first = list(new), list(past), first
        self.start = torch.tensor(np.concatenate([[0], np.cumsum(new)]) + first, dtype=torch.int32, device=device)
        self.pos0 = torch.tensor(list(past), dtype=torch.int32, device=device)
        self.rows, self.most = first + sum(new), max(new)

    def spans(self):
        at = self.first
        for s, (t, p) in enumerate(zip(self.new, self.past)):
            yield s, at, t, p
            at += t


def attention(cache, q, batch, theta, neox, window=0, scale=None):
    """[rows, n_head, hd] in 64 bits, over what the pools hold"""
    values = cache.values()
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    group = q.shape[1] // cache.n_kv
    for s, at, t, p in batch.spans():
        if t == 0:
            continue
        k, v = cache.rows(s, p + t, values)
        pos = torch.arange(p, p + t, device=q.device)
        x = turned(q[at:at + t], pos, theta, neox)
        key = torch.arange(p + t, device=q.device)
        seen = key <= pos[:, None]
        if window:
            seen &= key > pos[:, None] - window
        for h in range(q.shape[1]):
            w = (x[:, h] @ k[:, h // group].T) * (cache.hd ** -0.5 if scale is None else scale)
            w = torch.softmax(w.masked_fill(~seen, -float("inf")), -1)
            for i in range(t) if not torch.isfinite(v[:, h // group]).all() else ():
                out[at + i, h] = w[i, seen[i]] @ v[seen[i], h // group]
            if torch.isfinite(v[:, h // group]).all():
                out[at:at + t, h] = w @ v[:, h // group]
    return out
