"""Small plans over a paged cache for the tests of the operators for many conversations at once, and the operators'
definitions in 64 bits on the CPU (a row at a time, no code shared with the kernels)."""
import ctypes as C
import math

import numpy as np
import torch

from geode_b200 import batch as gb

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
CODE = {"f32": gb.F32, "bf16": gb.BF16, "f16": gb.F16, "i8": gb.I8}
HALF_STEP = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}   # of a rounding to nearest, relative


class Plan:
    """rows[s] new rows and lengths[s] positions of each sequence, pages in random order, unused table entries -1; the
    step's buffers hold `spare` rows more than the sequences own."""

    def __init__(self, rows, lengths, page, kv_heads, dim, cache, seed=0, head_major=False, spare=0, max_rows=None,
                 extra_pages=2, device="cuda", fill=None):
        rng = np.random.default_rng(seed)
        self.rows, self.lengths, self.page, self.cache, self.device = list(rows), list(lengths), page, cache, device
        self.n_rows = sum(rows) + spare
        self.width = max(1, max((n + page - 1) // page for n in lengths))
        need = sum((n + page - 1) // page for n in lengths)
        self.n_pages = need + extra_pages
        ids = rng.permutation(self.n_pages).astype(np.int32)
        table = np.full((len(rows), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(lengths):
            k = (n + page - 1) // page
            table[s, :k] = ids[at:at + k]
            at += k
        self.table_host = table
        self.start_host = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device)  # noqa: E731
        self.table, self.row_start = dev(table), dev(self.start_host)
        self.length = dev(np.array(lengths, np.int32))
        self.kv_heads, self.dim = kv_heads, dim
        shape = (self.n_pages, 2, kv_heads, page, dim) if head_major else (self.n_pages, 2, page, kv_heads, dim)
        self.buffer = torch.zeros(shape, dtype=TORCH[cache], device=device)
        self.scales = torch.zeros(shape[:4], device=device) if cache == "i8" else None
        if fill is not None:
            (self.buffer if self.scales is None else self.scales).fill_(fill)
        # [page][2][position][head][dim]
        self.view = self.buffer.transpose(2, 3) if head_major else self.buffer
        self.scale_view = None if self.scales is None else (self.scales.transpose(2, 3) if head_major else self.scales)
        v, s = self.view, self.scale_view
        st = (0, 0, 0, 0) if s is None else s.stride()
        self.kv = gb.PagedKV(k=v[:, 0].data_ptr(), v=v[:, 1].data_ptr(), k_scale=None if s is None else s[:, 0].data_ptr(),
                             v_scale=None if s is None else s[:, 1].data_ptr(), type=CODE[cache], n_pages=self.n_pages,
                             page_size=page, n_kv_heads=kv_heads, head_dim=dim, page_stride=v.stride(0),
                             pos_stride=v.stride(2), head_stride=v.stride(3), scale_page_stride=st[0],
                             scale_pos_stride=st[2], scale_head_stride=st[3])
        self.batch = gb.PagedBatch(n_seq=len(rows), n_rows=self.n_rows, max_rows=max_rows or max(1, max(rows)),
                                   max_pages=self.width, row_start=self.row_start.data_ptr(),
                                   length=self.length.data_ptr(), pages=self.table.data_ptr(),
                                   pages_stride=self.width)

    def places(self):
        """(row, sequence, position, page, offset) of every row of a sequence that has a position."""
        for s, n in enumerate(self.rows):
            for i in range(n):
                p = self.lengths[s] - n + i
                if p >= 0:
                    yield int(self.start_host[s]) + i, s, p, int(self.table_host[s, p // self.page]), p % self.page

    def randomize(self, seed):
        """Cache rows as a model leaves them; what no sequence holds: NaN scales or values."""
        g = torch.Generator().manual_seed(seed)
        n, P = self.n_pages, self.page
        if self.cache == "i8":
            codes = torch.randint(-127, 128, (n, 2, P, self.kv_heads, self.dim), generator=g, dtype=torch.int8)
            sc = (0.3 + torch.rand(n, 2, P, self.kv_heads, generator=g)) * 0.02
        else:
            codes = torch.randn(n, 2, P, self.kv_heads, self.dim, generator=g).to(TORCH[self.cache])
            sc = None
        held = torch.zeros(n, P, dtype=torch.bool)
        for s, length in enumerate(self.lengths):
            for p in range(length):
                held[self.table_host[s, p // P], p % P] = True
        out = ~held[:, None, :, None].expand(n, 2, P, self.kv_heads)
        if sc is None:
            codes = torch.where(out[..., None], torch.tensor(float("nan"), dtype=codes.dtype), codes)
        else:
            sc = torch.where(out, float("nan"), sc)
            self.scale_view.copy_(sc)
        self.view.copy_(codes)
        return codes, sc

    def values(self, s, which, upto):
        """The first `upto` positions' rows of sequence s in 64 bits: [position][head][dim]."""
        rows = []
        v = self.view.cpu()
        sc = None if self.scale_view is None else self.scale_view.cpu()
        for p in range(upto):
            at = (int(self.table_host[s, p // self.page]), which, p % self.page)
            x = v[at].double()
            rows.append(x if sc is None else x * sc[at].double()[:, None])
        return torch.stack(rows) if rows else torch.zeros(0, self.kv_heads, self.dim, dtype=torch.float64)


def norm_rotate(x, pos, w, eps, inv_freq):
    """One head vector in 64 bits (numpy): the zero-centred norm (w None: off), then rotate-half."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / math.sqrt((x * x).sum() / len(x) + eps) * (1.0 + np.asarray(w, np.float64))
    h = len(inv_freq)
    if h:
        a = pos * np.asarray(inv_freq, np.float64)
        lo, hi = x[:h].copy(), x[h:2 * h].copy()
        x = x.copy()
        x[:h], x[h:2 * h] = lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)
    return x


def codes_of(y):
    """int8 codes and scale of a row by the definition: from its 32-bit values, 127 y / amax to nearest even."""
    y = np.asarray(y, np.float32).astype(np.float64)
    top = np.abs(y).max()
    if top == 0:
        return np.zeros(len(y), np.int8), np.float32(0)
    return np.rint(y * 127.0 / top).astype(np.int8), np.float32(top / 127.0)


def attend(q, keys, values, scale):
    """One row's heads over the positions it sees: q [heads][dim], keys / values [position][kv head][dim] (64 bits).
    (out, lse, sum of p |v| per output, the largest sum of |q k| scale of a score)."""
    nh, hd = q.shape
    n, nkv = keys.shape[0], keys.shape[1]
    if n == 0:
        z = torch.zeros(nh, hd, dtype=torch.float64)
        return z, torch.full((nh,), -math.inf, dtype=torch.float64), z, torch.zeros(nh, dtype=torch.float64)
    g = nh // nkv
    s = torch.einsum("hgd,phd->hgp", q.view(nkv, g, hd), keys) * scale
    mag = torch.einsum("hgd,phd->hgp", q.view(nkv, g, hd).abs(), keys.abs()).amax(-1) * abs(scale)
    p = torch.softmax(s, -1)
    return (torch.einsum("hgp,phd->hgd", p, values).reshape(nh, hd), torch.logsumexp(s, -1).reshape(nh),
            torch.einsum("hgp,phd->hgd", p, values.abs()).reshape(nh, hd), mag.reshape(nh))


def adjust_row(x, V, history, drafts, rules, bias, mask_words):
    """One row of logits (float64 numpy) by the rules; rules = (repetition, frequency, presence)."""
    x = np.asarray(x, np.float64).copy()
    for t, b in dict((t, b) for t, b in bias if 0 <= t < V).items():
        x[t] += b
    seen = {}
    for t in list(history) + list(drafts):
        if 0 <= t < V:
            seen[t] = seen.get(t, 0) + 1
    r, f, p = rules
    for t, c in seen.items():
        x[t] = x[t] / r if x[t] > 0 else x[t] * r
        x[t] = x[t] - f * c - p
    if mask_words is not None:
        v = np.arange(V)
        x[((mask_words[v >> 5].astype(np.int64) >> (v & 31)) & 1) == 0] = -np.inf
    return x


def ref(s):
    return C.byref(s)
