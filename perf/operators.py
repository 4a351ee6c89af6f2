"""What the operators for many conversations at once are measured on: rows appended to a paged key-value cache (head
norms, rotary positions and the cache's rounding on the way), the attention of each sequence's newest rows over that
cache, and the logits' penalties, biases and grammar masks in front of the acceptance.

Where `own` is false `run` computes them in elementary torch operations, where it is true through the package's C entry
points. Rows are ragged: sequence s owns rows row_start[s] .. row_start[s + 1] of the step's buffers, its cache holds
length[s] positions (those rows included) and its pages are listed in a table."""
import ctypes
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
CODE = {"f32": 0, "bf16": 1, "f16": 2, "i8": 3}   # the entry points' type codes
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}


# ------------------------------------------------------------------------------------------------ the cases ----
def _append(name, act, cache, heads, kv_heads, dim, rope, norm, seqs, rows, context, page, ragged=False, head_major=False):
    return dict(name=name, op="append", act=act, cache=cache, heads=heads, kv_heads=kv_heads, dim=dim, rope=rope, norm=norm,
                seqs=seqs, rows=rows, context=context, page=page, ragged=ragged, head_major=head_major)


def _attend(name, act, cache, heads, kv_heads, dim, seqs, rows, context, page, ragged=False, head_major=False, window=0):
    return dict(name=name, op="attend", act=act, cache=cache, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs, rows=rows,
                context=context, page=page, ragged=ragged, head_major=head_major, window=window)


def _adjust(name, act, seqs, drafts, vocab, history, biases, masked):
    return dict(name=name, op="adjust", act=act, seqs=seqs, drafts=drafts, vocab=vocab, history=history, biases=biases,
                masked=masked)


def listed():
    return [
        # one conversation, one new token: the launch and its latency are what it costs
        _append("append_one", "f32", "i8", 16, 2, 256, 64, True, 1, 1, 8192, 64),
        # a verify step of 256 conversations, five rows each, into the engine's int8 cache
        _append("append_verify", "f32", "i8", 16, 2, 256, 64, True, 256, 5, 4096, 64),
        # prompts of uneven lengths in 16-bit rows, every dimension rotated, no head norms
        _append("append_prompts", "bf16", "bf16", 32, 8, 128, 128, False, 7, 4099, 4500, 16, ragged=True),
        # the same from 16-bit activations into the int8 cache, heads outermost within a page
        _append("append_prompts_i8", "f16", "i8", 32, 4, 128, 128, True, 5, 3001, 6000, 32, ragged=True, head_major=True),
        # one conversation's next token at the benchmark's context
        _attend("attend_one", "f32", "i8", 16, 2, 256, 1, 1, 8192, 64),
        # a decoding batch, lengths all over the range
        _attend("attend_batch", "bf16", "i8", 16, 2, 256, 64, 1, 8192, 64, ragged=True),
        # a verify step: the accepted token and up to four drafts of each conversation, 32-bit activations
        _attend("attend_verify", "f32", "i8", 16, 2, 256, 32, 5, 8192, 64, ragged=True),
        # few very long conversations
        _attend("attend_long", "bf16", "bf16", 16, 2, 256, 2, 1, 131072, 64, ragged=True),
        # many short ones: small pages, four query heads to a key head
        _attend("attend_short", "f16", "f16", 32, 8, 128, 128, 1, 1000, 16, ragged=True, head_major=True),
        # one conversation's next token: a grammar mask, a history and some biases
        _adjust("adjust_one", "f32", 1, 0, 248320, 2000, 40, True),
        # a verify step of 64 conversations, four drafts each
        _adjust("adjust_verify", "f32", 64, 4, 248320, 4000, 100, True),
        # 16-bit logits of an odd vocabulary
        _adjust("adjust_bf16", "bf16", 100, 0, 50257, 1500, 300, True),
    ]


def _unnamed(c):
    del c["name"]
    return c


def _spread(rng, low, high):
    """A whole number from low to high, evenly over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "adjust"])
    if op == "adjust":
        act, k = rng.choice(["f32", "f32", "bf16", "f16"]), rng.choice([0, 0, 1, 3, 4, 8])
        vocab = _spread(rng, 997, 260000)
        most = max(1, min(512, 64 * 5 * 248320 // ((k + 1) * vocab)))
        return _unnamed(_adjust("", act, _spread(rng, 1, most), k, vocab, _spread(rng, 1, 8000), rng.choice([0, 1, 17, 300]),
                                rng.random() < 0.7))
    dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    act, cache = rng.choice([("f32", "i8"), ("bf16", "i8"), ("f16", "i8"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
    page, head_major, ragged = rng.choice([16, 32, 64, 100, 128]), rng.random() < 0.4, rng.random() < 0.7
    if op == "append":
        rows = rng.choice([1, 1, 2, 5, 8, 0])
        rows = rows or _spread(rng, 9, 4000)
        seqs = _spread(rng, 1, max(1, min(256, 500_000_000 // (rows * heads * dim * 2 * SIZE[act]))))
        context = rows + _spread(rng, 1, 20000)
        while seqs * context * kv_heads * dim > 256 * 4096 * 2 * 256:
            context = rows + (context - rows) // 2
            seqs = max(1, seqs // 2)
        return _unnamed(_append("", act, cache, heads, kv_heads, dim, rng.choice([dim, dim // 2, dim // 4]),
                                rng.random() < 0.5, seqs, rows, context, page, ragged, head_major))
    rows = rng.choice([1, 1, 1, 2, 3, 5, 8])
    seqs = _spread(rng, 1, 128)
    context = rows + _spread(rng, 1, 60000)
    while seqs * context * kv_heads * dim * (rows + 1) * SIZE[cache] > 2 * 64 * 8192 * 2 * 256:
        if seqs > 1 and rng.random() < 0.5:
            seqs -= seqs // 2
        else:
            context = max(rows, context - context // 2)
    return _unnamed(_attend("", act, cache, heads, kv_heads, dim, seqs, rows, context, page, ragged, head_major,
                            rng.choice([0, 0, 0, 500])))


# ------------------------------------------------------------------------------------------- plans and inputs ----
def _counts(c):
    """Each sequence's rows and positions: every sequence alike, or spread over the range (golden-ratio steps)."""
    S, T, L = c["seqs"], c["rows"], c["context"]
    if not c["ragged"]:
        return [T] * S, [L] * S
    rows = [max(1, math.ceil(T * ((0.5 + 0.7548776662 * i) % 1.0))) for i in range(S)]
    return rows, [max(r, math.ceil(L * ((0.9 + 0.6180339887 * i) % 1.0))) for i, r in enumerate(rows)]


def _paged(c, g):
    """The batch's plan and its cache: pages in no order, a few of them nobody's."""
    rows, lengths = _counts(c)
    S, P = c["seqs"], c["page"]
    order = torch.randperm(S, generator=torch.Generator().manual_seed(g.initial_seed())).tolist()
    rows, lengths = [rows[i] for i in order], [lengths[i] for i in order]
    width = (max(lengths) + P - 1) // P
    need = [(n + P - 1) // P for n in lengths]
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    need_t, first = torch.tensor(need, device="cuda"), torch.tensor([0] + need[:-1], device="cuda").cumsum(0)
    col = torch.arange(width, device="cuda")
    table = torch.where(col < need_t[:, None], ids[(first[:, None] + col).clamp(max=n_pages - 1)], -1).to(torch.int32)
    start = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
    s = {"case": c, "n_rows": sum(rows), "width": width, "n_pages": n_pages, "table": table.contiguous(), "row_start": start,
         "max_rows": max(rows), "length": torch.tensor(lengths, device="cuda", dtype=torch.int32)}
    shape = (n_pages, 2, c["kv_heads"], P, c["dim"]) if c["head_major"] else (n_pages, 2, P, c["kv_heads"], c["dim"])
    s["kv"] = torch.zeros(shape, dtype=TYPES[c["cache"]], device="cuda")
    s["scale"] = torch.zeros(shape[:4], device="cuda") if c["cache"] == "i8" else None
    # the row's sequence, its position, and where that lies
    s["seq_of"] = torch.repeat_interleave(torch.arange(S, device="cuda"), torch.tensor(rows, device="cuda"))
    s["row_in"] = torch.arange(s["n_rows"], device="cuda") - start[s["seq_of"]]
    s["position"] = s["length"][s["seq_of"]].long() - torch.tensor(rows, device="cuda")[s["seq_of"]] + s["row_in"]
    s["at_page"] = s["table"][s["seq_of"], s["position"] // P].long()
    s["at_offset"] = s["position"] % P
    return s


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    if c["op"] == "adjust":
        S, k, V = c["seqs"], c["drafts"], c["vocab"]
        T = k + 1
        s = {"case": c, "logits": (3.0 * normal(S * T, V)).to(TYPES[c["act"]])}
        s["out"] = torch.empty_like(s["logits"])
        H = max(1, c["history"])
        # tokens come back as words do: small ids often, large ones seldom
        zipf = lambda *n: ((V + 1.0) ** torch.rand(*n, generator=g, device="cuda") - 1).long().clamp(0, V - 1).to(torch.int32)  # noqa: E731
        s["history"] = zipf(S, H)
        s["history_len"] = torch.ceil(H * ((torch.arange(S, device="cuda") * 0.6180339887 + 0.9) % 1.0)).to(torch.int32)
        s["drafts"] = zipf(S, max(1, k))
        s["repetition"] = 1.0 + 0.3 * torch.rand(S, generator=g, device="cuda")
        s["frequency"] = 0.4 * torch.rand(S, generator=g, device="cuda")
        s["presence"] = 1.5 * torch.rand(S, generator=g, device="cuda")
        B = max(1, c["biases"])
        s["bias_id"] = torch.randint(0, V, (S, B), generator=g, device="cuda", dtype=torch.int32)
        s["bias"] = 5.0 * normal(S, B)
        s["bias_len"] = torch.full((S,), c["biases"], device="cuda", dtype=torch.int32)
        words = (V + 31) // 32
        M = max(1, S * T // 2)   # half of the rows are under a grammar, each in a state of its own
        bits = lambda: torch.randint(-2**31, 2**31 - 1, (M, words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)  # noqa: E731
        s["mask"] = bits() & bits()
        pick = torch.full((S * T,), -1, device="cuda", dtype=torch.int32)
        if c["masked"]:
            pick[torch.randperm(S * T, generator=g, device="cuda")[:M]] = torch.arange(M, device="cuda", dtype=torch.int32)
        s["mask_row"] = pick
        return s
    s = _paged(c, g)
    act, N, nh, nkv, hd = TYPES[c["act"]], s["n_rows"], c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "append":
        s["q"], s["k"], s["v"] = normal(N, nh, hd).to(act), normal(N, nkv, hd).to(act), normal(N, nkv, hd).to(act)
        s["q_out"] = torch.empty_like(s["q"])
        s["q_norm"], s["k_norm"] = 0.1 * normal(hd), 0.1 * normal(hd)
        s["inv_freq"] = (1.0e7 ** (-torch.arange(0, c["rope"], 2, device="cuda", dtype=torch.float64) / c["rope"])).float()
        s["eps"] = 1e-6
        return s
    s["q"] = (1.5 * normal(N, nh, hd)).to(act)
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(N, nh, device="cuda")
    if c["cache"] == "i8":
        s["kv"].copy_(torch.randint(-127, 128, s["kv"].shape, generator=g, device="cuda", dtype=torch.int8))
        s["scale"].copy_((0.5 + torch.rand(s["scale"].shape, generator=g, device="cuda")) * (1.7 / 127))
    else:
        s["kv"].normal_(generator=g)
    s["softmax_scale"] = 1.0 / math.sqrt(hd)
    return s


# ------------------------------------------------------------------------------------------------ the calls ----
def _bind(s):
    """The entry points' descriptors of the state's buffers: a program fills them where it allocates those."""
    from geode_b200 import batch as gb
    from geode_b200 import cuda_lib

    c, d = s["case"], {}
    d["lib"] = lib = cuda_lib()
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if c["op"] == "adjust":
        d["rules"] = gb.LogitRules(
            history=ptr(s["history"]), history_len=ptr(s["history_len"]), history_stride=s["history"].stride(0),
            drafts=ptr(s["drafts"]) if c["drafts"] else None, repetition=ptr(s["repetition"]), frequency=ptr(s["frequency"]),
            presence=ptr(s["presence"]), bias_id=ptr(s["bias_id"]), bias=ptr(s["bias"]), bias_len=ptr(s["bias_len"]),
            bias_stride=s["bias"].stride(0), mask=ptr(s["mask"]), mask_row=ptr(s["mask_row"]), n_masks=s["mask"].shape[0],
            mask_stride=s["mask"].stride(0))
        d["refs"] = (ctypes.byref(d["rules"]),)
        return d
    view = s["kv"].transpose(2, 3) if c["head_major"] else s["kv"]   # [page][2][position][head][dim]
    scale = None if s["scale"] is None else s["scale"].transpose(2, 3) if c["head_major"] else s["scale"]
    st = (0, 0, 0, 0) if scale is None else scale.stride()
    d["kv"] = gb.PagedKV(
        k=view[:, 0].data_ptr(), v=view[:, 1].data_ptr(), k_scale=None if scale is None else scale[:, 0].data_ptr(),
        v_scale=None if scale is None else scale[:, 1].data_ptr(), type=CODE[c["cache"]], n_pages=s["n_pages"],
        page_size=c["page"], n_kv_heads=c["kv_heads"], head_dim=c["dim"], page_stride=view.stride(0),
        pos_stride=view.stride(2), head_stride=view.stride(3), scale_page_stride=st[0], scale_pos_stride=st[2],
        scale_head_stride=st[3])
    d["batch"] = gb.PagedBatch(
        n_seq=c["seqs"], n_rows=s["n_rows"], max_rows=s["max_rows"], max_pages=s["width"], row_start=ptr(s["row_start"]),
        length=ptr(s["length"]), pages=ptr(s["table"]), pages_stride=s["table"].stride(0))
    if c["op"] == "append":
        d["rows"] = gb.AppendRows(
            type=CODE[c["act"]], n_heads=c["heads"], q=ptr(s["q"]), k=ptr(s["k"]), v=ptr(s["v"]), q_out=ptr(s["q_out"]),
            q_stride=s["q"].stride(0), q_head_stride=s["q"].stride(1), k_stride=s["k"].stride(0), v_stride=s["v"].stride(0),
            q_out_stride=s["q_out"].stride(0), q_norm=ptr(s["q_norm"]) if c["norm"] else None,
            k_norm=ptr(s["k_norm"]) if c["norm"] else None, eps=s["eps"], rope_dim=c["rope"], inv_freq=ptr(s["inv_freq"]))
    else:
        d["rows"] = gb.AttnRows(
            type=CODE[c["act"]], n_heads=c["heads"], q=ptr(s["q"]), out=ptr(s["out"]), lse=ptr(s["lse"]),
            q_stride=s["q"].stride(0), q_head_stride=s["q"].stride(1), out_stride=s["out"].stride(0),
            scale=s["softmax_scale"], window=c["window"])
        d["bytes"] = lib.gcuda_op_paged_attn_work_bytes(ctypes.byref(d["kv"]), ctypes.byref(d["batch"]), c["heads"])
        d["work"] = torch.empty(d["bytes"], dtype=torch.uint8, device="cuda")
    d["refs"] = tuple(ctypes.byref(d[x]) for x in ("kv", "batch", "rows"))
    return d


def _check(rc):
    if rc != 0:
        raise RuntimeError(f"entry point: {rc}")


def _own(s):
    if "bound" not in s:
        s["bound"] = _bind(s)
    d, c, stream = s["bound"], s["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        _check(d["lib"].gcuda_op_paged_append(*d["refs"], stream))
    elif c["op"] == "attend":
        _check(d["lib"].gcuda_op_paged_attn(*d["refs"], d["work"].data_ptr(), d["bytes"], stream))
    else:
        _check(d["lib"].gcuda_op_logits_adjust(*d["refs"], s["logits"].data_ptr(), s["out"].data_ptr(), CODE[c["act"]],
                                               c["seqs"], c["drafts"], c["vocab"], s["logits"].stride(0),
                                               s["out"].stride(0), stream))


# ------------------------------------------------------------------------------------------ the plain forms ----
def _normed(x, w, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * (1.0 + w.to(x.dtype))


def _rotated(x, position, inv_freq):
    angle = position.double()[:, None, None] * inv_freq.double()   # far positions: the angle in 64 bits
    cos, sin = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
    h = inv_freq.numel()
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


def _plain_append(s):
    c = s["case"]
    q, k, v = s["q"].float(), s["k"], s["v"]
    k = k.double() if c["cache"] == "i8" else k.float()   # codes next to a border: in 64 bits
    if c["norm"]:
        q, k = _normed(q, s["q_norm"], s["eps"]), _normed(k, s["k_norm"], s["eps"])
    s["q_out"].copy_(_rotated(q, s["position"], s["inv_freq"]))
    k = _rotated(k, s["position"], s["inv_freq"])
    both = torch.stack([k.float(), v.float()], 1)   # [row][2][head][dim]
    kv = s["kv"].transpose(2, 3) if c["head_major"] else s["kv"]
    which = torch.arange(2, device="cuda")
    at = (s["at_page"][:, None], which, s["at_offset"][:, None])
    if c["cache"] == "i8":
        most = both.abs().amax(-1, keepdim=True)
        codes = torch.where(most > 0, torch.round(both.double() * 127.0 / most.double().clamp(min=1e-300)), 0.0)
        kv[at] = codes.to(torch.int8)
        (s["scale"].transpose(2, 3) if c["head_major"] else s["scale"])[at] = (most[..., 0].double() / 127.0).float()
    else:
        kv[at] = both.to(kv.dtype)


def _plain_attend(s):
    c = s["case"]
    S, P, nh, nkv, hd = c["seqs"], c["page"], c["heads"], c["kv_heads"], c["dim"]
    T, G, L = s["max_rows"], nh // nkv, s["width"] * P
    kv = (s["kv"].transpose(2, 3) if c["head_major"] else s["kv"])[s["table"].clamp(min=0).long()].float()
    if c["cache"] == "i8":
        kv = kv * (s["scale"].transpose(2, 3) if c["head_major"] else s["scale"])[s["table"].clamp(min=0).long()][..., None]
    k, v = (kv[:, :, i].reshape(S, L, nkv, hd).transpose(1, 2) for i in (0, 1))   # [sequence][head][position][dim]
    q = torch.zeros(S, T, nkv, G, hd, device="cuda")
    q[s["seq_of"], s["row_in"]] = s["q"].float().reshape(-1, nkv, G, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(S, nkv, T * G, hd)
    scores = (q @ k.transpose(2, 3)).reshape(S, nkv, T, G, L) * s["softmax_scale"]
    at = torch.arange(L, device="cuda")
    rows = s["row_start"][1:] - s["row_start"][:-1]
    last = (s["length"] - rows)[:, None] + torch.arange(T, device="cuda")   # the position of each row
    seen = at <= last[..., None]
    if c["window"]:
        seen &= at > last[..., None] - c["window"]
    scores = torch.where(seen[:, None, :, None], scores, -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - most)
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(S, nkv, T * G, L) @ v).reshape(S, nkv, T, G, hd) / total
    lse = (most + total.log())[..., 0]
    s["out"].copy_(o.permute(0, 2, 1, 3, 4)[s["seq_of"], s["row_in"]].reshape(-1, nh, hd))
    s["lse"].copy_(lse.permute(0, 2, 1, 3)[s["seq_of"], s["row_in"]].reshape(-1, nh))


def _plain_adjust(s):
    c = s["case"]
    S, k, V = c["seqs"], c["drafts"], c["vocab"]
    T, H, B = k + 1, s["history"].shape[1], s["bias"].shape[1]
    x = s["logits"].float().reshape(S, T, V)
    if c["biases"]:
        # of a token's entries the last one counts
        place = torch.arange(1, B + 1, device="cuda").expand(S, B)
        place = torch.where(place <= s["bias_len"][:, None], place, 0)
        last = torch.zeros(S, V, dtype=torch.long, device="cuda").scatter_reduce(1, s["bias_id"].long(), place, "amax")
        x = x + torch.where(last > 0, s["bias"].gather(1, (last - 1).clamp(min=0)), 0.0)[:, None]
    live = (torch.arange(H, device="cuda") < s["history_len"][:, None]).int()
    count = torch.zeros(S, V, dtype=torch.int32, device="cuda").scatter_add_(1, s["history"].long(), live)
    count = count[:, None].expand(S, T, V)
    if k:
        before = torch.ones(T, k, dtype=torch.int32, device="cuda").tril(-1).expand(S, T, k)   # row i has drafts 0 .. i - 1
        count = count.contiguous().scatter_add_(2, s["drafts"].long()[:, None].expand(S, T, k), before)
    r, f, p = (s[n][:, None, None] for n in ("repetition", "frequency", "presence"))
    x = torch.where(count > 0, torch.where(x > 0, x / r, x * r) - f * count - p, x).reshape(S * T, V)
    if c["masked"]:
        v = torch.arange(V, device="cuda")
        allowed = (s["mask"][:, v >> 5] >> (v & 31).int() & 1).bool()
        x = torch.where((s["mask_row"] >= 0)[:, None] & ~allowed[s["mask_row"].clamp(min=0).long()], -math.inf, x)
    s["out"].copy_(x)


def run(state):
    s = state
    if own:
        _own(s)
    else:
        {"append": _plain_append, "attend": _plain_attend, "adjust": _plain_adjust}[s["case"]["op"]](s)
    return _answer(s)


def _answer(s):
    c = s["case"]
    if c["op"] == "adjust":
        return {"logits": s["out"]}
    if c["op"] == "attend":
        return {"out": s["out"], "lse": s["lse"]}
    # what the cache now holds for the appended rows, as values
    at = (s["at_page"], slice(None), s["at_offset"])
    held = (s["kv"].transpose(2, 3) if c["head_major"] else s["kv"])[at]
    if c["cache"] == "i8":
        held = held * (s["scale"].transpose(2, 3) if c["head_major"] else s["scale"])[at][..., None]
    return {"q": s["q_out"], "kv": held}


# ---------------------------------------------------------------------------------------------------- work ----
def work(case):
    c = case
    if c["op"] == "adjust":
        rows = c["seqs"] * (c["drafts"] + 1)
        n = rows * c["vocab"]
        return {"bytes": 2 * n * SIZE[c["act"]] + (max(1, rows // 2) * c["vocab"] / 8 if c["masked"] else 0)
                + c["seqs"] * (2 * c["history"] + 8 * c["biases"]), "flops": 2 * n}
    rows, lengths = _counts(c)
    N, nh, nkv, hd = sum(rows), c["heads"], c["kv_heads"], c["dim"]
    held = 2 * nkv * (hd * SIZE[c["cache"]] + (4 if c["cache"] == "i8" else 0))
    if c["op"] == "append":
        return {"bytes": N * ((2 * nh + 2 * nkv) * hd * SIZE[c["act"]] + held), "flops": 8 * N * (nh + 2 * nkv) * hd}
    w = c["window"] or 1 << 40
    read = sum(min(n, w + t - 1) for t, n in zip(rows, lengths))
    pairs = sum(min(n - t + i + 1, w) for t, n in zip(rows, lengths) for i in range(t))
    return {"bytes": read * held + N * nh * (2 * hd * SIZE[c["act"]] + 4), "flops": 4 * hd * nh * pairs}


# --------------------------------------------------------------------------------------------------- exact ----
def exact(case, seed):
    """The same from the definitions in 64 bits, a sequence at a time."""
    s, c = prepare(case, seed), case
    return {"append": _exact_append, "attend": _exact_attend, "adjust": _exact_adjust}[c["op"]](s, c)


def _exact_append(s, c):
    hd, half = c["dim"], c["rope"] // 2

    def vectors(x, w):
        x = x.to(torch.float64)
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / hd + s["eps"]).sqrt() * (w.to(torch.float64) + 1)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.outer(s["position"].to(torch.float64), s["inv_freq"].to(torch.float64)))[:, None]
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], dim=-1)

    q = vectors(s["q"], s["q_norm"] if c["norm"] else None)
    held = torch.stack([vectors(s["k"], s["k_norm"] if c["norm"] else None), s["v"].to(torch.float64)], dim=1)
    if c["cache"] == "i8":
        # the rows as 32-bit values, then the nearest of 255 steps (the even one of two)
        held = held.to(torch.float32).to(torch.float64)
        top = held.abs().max(dim=-1, keepdim=True).values
        codes = (held * 127 / top).round()
        held = torch.where(top > 0, codes * (top / 127), torch.zeros_like(held))
    return {"q": q, "kv": held}


def _exact_attend(s, c):
    nh, nkv, hd = c["heads"], c["kv_heads"], c["dim"]
    out = torch.zeros(s["n_rows"], nh, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((s["n_rows"], nh), -math.inf, dtype=torch.float64, device="cuda")
    start, length = s["row_start"].tolist(), s["length"].tolist()
    for i, n in enumerate(length):
        ids = s["table"][i, : -(-n // c["page"])].long()
        block = s["kv"][ids].to(torch.float64)
        if s["scale"] is not None:
            block *= s["scale"][ids].to(torch.float64)[..., None]
        if c["head_major"]:
            block = block.permute(0, 1, 3, 2, 4)
        keys, values = (block[:, j].flatten(0, 1)[:n] for j in (0, 1))
        for t in range(start[i], start[i + 1]):
            end = n - (start[i + 1] - t) + 1
            begin = max(0, end - c["window"]) if c["window"] else 0
            if end <= begin:
                continue
            query = s["q"][t].to(torch.float64).view(nkv, nh // nkv, hd)
            weight = torch.einsum("hgd,phd->hgp", query, keys[begin:end]) * s["softmax_scale"]
            lse[t] = torch.logsumexp(weight, dim=-1).flatten()
            out[t] = torch.einsum("hgp,phd->hgd", torch.softmax(weight, dim=-1), values[begin:end]).reshape(nh, hd)
    return {"out": out, "lse": lse}


def _exact_adjust(s, c):
    S, T, V = c["seqs"], c["drafts"] + 1, c["vocab"]
    out = s["logits"].to(torch.float64)
    word = torch.arange(V, device="cuda") // 32
    bit = torch.arange(V, device="cuda") % 32
    for i in range(S):
        n, b = int(s["history_len"][i]), int(s["bias_len"][i])
        last = dict(zip(s["bias_id"][i, :b].tolist(), s["bias"][i, :b].tolist()))
        ids = torch.tensor(list(last), dtype=torch.long, device="cuda")
        plus = torch.tensor(list(last.values()), dtype=torch.float64, device="cuda")
        said = s["history"][i, :n].long()
        r, f, p = (float(s[x][i]) for x in ("repetition", "frequency", "presence"))
        for t in range(T):
            row = out[i * T + t]
            row[ids] += plus
            tokens, times = torch.cat([said, s["drafts"][i, :t].long()]).unique(return_counts=True)
            x = row[tokens]
            row[tokens] = torch.where(x > 0, x / r, x * r) - f * times - p
            m = int(s["mask_row"][i * T + t])
            if m >= 0:
                row[(s["mask"][m][word].long() >> bit & 1) == 0] = -math.inf
    return {"logits": out}
