"""The key/value cache of a language model as an index of this library: what is measured, and its plain forms.

A cache holds the keys and values of many sequences in pages (`table[b, i]`: the page of block i of sequence b), in 16
bits, or in 8 bits with one scale for each row of a head, and for every block the componentwise bounds of its keys.  Four
operators work on it: `add` writes new rows (rounding them to 8 bits) and keeps the bounds, `vectors` reads rows back,
`search_blocks` finds for every query the blocks whose bounds promise the largest inner products, and `attend` is
attention over the blocks found, or over all of them.  The last rows of sequence b are the ones that a call is about: row
i of its n rows stands at position lens[b] - n + i.
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOP = {"int8": 127.0, "e4m3": 448.0}  # the largest value that each 8-bit type holds


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of a server with 24 requests: a row each
        dict(name="add_token", path="add", kind="int8", dtype="bf16", B=24, new=1, ctx=4000, page=64, heads=8, group=4, dim=128),
        # the prompts of six requests, of different lengths, at once
        dict(name="add_prompts", path="add", kind="e4m3", dtype="bf16", B=6, new=2900, ctx=2900, page=64, heads=8, group=4, dim=128),
        # the rows of one short sequence, to move them to another cache; heads of 96
        dict(name="vectors_short", path="vectors", kind="int8", dtype="fp16", B=1, new=777, ctx=777, page=16, heads=4, group=3, dim=96),
        # long sequences read back whole, for an attention that wants plain rows
        dict(name="vectors_long", path="vectors", kind="e4m3", dtype="bf16", B=4, new=30000, ctx=30000, page=64, heads=8, group=4, dim=128),
        # a decoding step of one request with a long document before it
        dict(name="search_one", path="search", kind="int8", dtype="bf16", B=1, new=1, ctx=130000, page=64, heads=8, group=4, dim=128, k=32),
        # a decoding step of 48 requests, smaller blocks, seven query heads to a key head
        dict(name="search_batch", path="search", kind="e4m3", dtype="fp16", B=48, new=1, ctx=16000, page=32, heads=4, group=7, dim=128, k=64),
        # a piece of two prompts, each query with blocks of its own
        dict(name="search_prompt", path="search", kind="same", dtype="bf16", B=2, new=1900, ctx=33000, page=64, heads=8, group=4, dim=128, k=24),
        # attention of the same single request over the blocks found
        dict(name="attend_one", path="attend", kind="same", dtype="bf16", B=1, new=1, ctx=50000, page=64, heads=8, group=4, dim=128, k=32),
        # a full batch's decoding step over an 8-bit cache
        dict(name="attend_batch", path="attend", kind="int8", dtype="bf16", B=64, new=1, ctx=20000, page=64, heads=8, group=8, dim=128, k=48),
        # a decoding step over whole sequences: nothing selected
        dict(name="attend_all", path="attend", kind="e4m3", dtype="fp16", B=12, new=1, ctx=15000, page=64, heads=8, group=4, dim=128, k=0),
        # four drafted tokens and the last one, each head its own keys, small blocks, heads of 64
        dict(name="attend_draft", path="attend", kind="same", dtype="fp16", B=7, new=5, ctx=5000, page=16, heads=12, group=1, dim=64, k=40),
        # a piece of two prompts over the blocks that each of its queries selected
        dict(name="attend_prompt", path="attend", kind="same", dtype="bf16", B=2, new=1000, ctx=17000, page=64, heads=8, group=4, dim=128, k=16),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    path = rng.choice(["add", "vectors", "search", "attend", "attend", "attend"])
    case = dict(path=path, kind=rng.choice(["same", "int8", "e4m3"]), dtype=rng.choice(["bf16", "fp16"]), heads=rng.choice([1, 2, 4, 8, 8]),
                dim=rng.choice([64, 96, 128, 128]), page=rng.choice([16, 32, 64, 64, 128]))
    case["group"] = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    row = case["heads"] * case["dim"]
    if path in ("add", "vectors"):
        case["new"] = rng.choice([1, _log(rng, 1, 20_000)])
        case["B"] = _log(rng, 1, max(1, min(256, 16_000_000 // (row * case["new"]))))
        case["ctx"] = case["new"] if path == "vectors" else case["new"] + rng.choice([0, _log(rng, 1, 2000)])
        case["B"] = max(1, min(case["B"], 60_000_000 // (row * case["ctx"])))
        return case
    case["new"] = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 1000)])
    case["ctx"] = case["new"] + _log(rng, 1, 60_000)
    dense = path == "attend" and rng.random() < 0.3
    case["k"] = 0 if dense else max(2, min(_log(rng, 4, 64), 3000 // case["page"]))
    if dense:
        case["new"] = min(case["new"], 250)
    case["B"] = max(1, min(_log(rng, 1, 64), 250_000_000 // (row * case["ctx"])))
    if case["new"] > 1:  # the plain form takes every query's blocks out of the cache by themselves
        seen = case["ctx"] if dense else case["k"] * case["page"]
        case["new"] = max(2, min(case["new"], 800_000_000 // (case["B"] * row * seen), 1_000_000_000 // (case["B"] * case["heads"] * case["group"] * seen)))
    return case


def _lengths(case):
    """Rows of this call and whole lengths of the sequences, none like its neighbour where there are several."""
    new = [max(1, case["new"] * (16 - (b * 23) % 9) // 16) for b in range(case["B"])]
    lens = [n + (case["ctx"] - case["new"]) * (16 - (b * 37) % 11) // 16 for b, n in enumerate(new)]
    return new, lens


# --------------------------------------------------------------------------------------------------------- inputs
def _first(x):
    """Where each of the numbers x begins when they stand one behind the other."""
    return [sum(x[:i]) for i in range(len(x) + 1)]


def prepare(case, seed):
    """Keys as they are met: some channels far from zero, the rows of a block like one another, queries that look for a few
    blocks and for the same ones over some positions."""
    g = torch.Generator("cuda")
    g.manual_seed(int(seed))
    rand = lambda *n: torch.rand(n, generator=g, device="cuda")  # noqa: E731
    randn = lambda *n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    dtype, kind, page, H, G, D, B = DTYPES[case["dtype"]], case["kind"], case["page"], case["heads"], case["group"], case["dim"], case["B"]
    new, lens = _lengths(case)
    blocks = [-(-n // page) for n in lens]
    W, P, T = max(blocks), sum(blocks) + 3, sum(new)
    at = _first(blocks)
    of = torch.randperm(P, generator=g, device="cuda").to(torch.int32)  # pages are handed out in no order
    table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(blocks):
        table[b, :n] = of[at[b] : at[b] + n]
    centre, channel = randn(P, H, D), 2.0 * randn(H, D) * (rand(H, D) < 0.1)
    k = ((centre[:, :, None] * 0.8 + channel[:, None]) + randn(P, H, page, D) * 0.6).to(dtype)
    v = (randn(P, H, page, D) + 0.3 * centre[:, :, None]).to(dtype)
    s = dict(case=case, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), cu=None)
    if case["new"] > 1 or case["path"] == "vectors":
        s["cu"] = torch.tensor(_first(new), dtype=torch.int32, device="cuda")
    bounds = torch.stack((k.amin(2), k.amax(2)), 2)
    codes, scale = _coded(bounds.flatten(2), "int8")
    pool = dict(k=k, v=v, k_scale=None, v_scale=None, bounds=bounds, bound_codes=codes.view(bounds.shape), bound_scale=scale)
    if kind != "same":
        pool["k"], pool["k_scale"] = _coded(k, kind)
        pool["v"], pool["v_scale"] = _coded(v, kind)
    s["pool"] = pool
    del k, v
    seq, pos = _places(s, T)
    # queries, and new keys and values, are parts of one projection's rows
    rows = randn(T, H * (G + 2), D) * 0.7
    run_of = torch.randint(0, 1 << 20, (B, max(new) // 32 + 2, 4), generator=g, device="cuda")[seq, (pos - pos[0]).clamp(min=0) // 32 % (max(new) // 32 + 2)]
    focus = centre[table[seq[:, None], run_of % (pos // page + 1)[:, None]].long()].mean(1)  # (T, H, D)
    rows.view(T, H * (G + 2), D)[:, : H * G] += (1.2 * focus)[:, :, None].expand(T, H, G, D).reshape(T, H * G, D)
    rows[:, H * G : H * (G + 1)] += channel
    s["rows"] = rows.to(dtype)
    s["q"], s["new_k"], s["new_v"] = s["rows"].split([H * G, H, H], 1)
    if case["path"] == "attend":
        s["blocks"] = _search(s, case["k"]) if case["k"] else None
    if own:  # the handle that a program keeps
        import ferrolm_b200 as fv

        s["cache"] = fv.KvCache(P, H, D, page_size=page, dtype=dtype, kind=kind, buffers=pool)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _places(s, T):
    """(sequence, position) of the T rows of a call."""
    lens = s["lens"].long()
    if s["cu"] is None:
        return torch.arange(T, device="cuda"), lens - 1
    cu, t = s["cu"].long(), torch.arange(T, device="cuda")
    seq = torch.bucketize(t, cu[1:], right=True)
    return seq, lens[seq] - cu[seq + 1] + t


def _coded(x, kind):
    """Rows in 8 bits: the largest absolute value stands for the type's largest.  The quotient lies next to the border of two
    codes too often for 32 bits; a row with a value that is not finite has the scale NaN and codes of zero."""
    top = TOP[kind]
    most = x.float().abs().amax(-1, keepdim=True)
    fine = torch.isfinite(most)
    scale = torch.where(fine, most / torch.full_like(most, top), torch.nan).squeeze(-1)
    y = torch.where(fine & (most > 0), x.double() * top / most.double(), 0.0)
    return (y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)), scale


def _add(s):
    pool, page = s["pool"], s["case"]["page"]
    k, v, kind = s["new_k"], s["new_v"], s["case"]["kind"]
    seq, pos = _places(s, k.shape[0])
    at, slot = s["table"][seq, pos // page].long(), pos % page
    if kind == "same":
        pool["k"][at, :, slot], pool["v"][at, :, slot] = k, v
    else:
        codes, scale = _coded(k, kind)
        pool["k"][at, :, slot], pool["k_scale"][at, :, slot] = codes, scale
        codes, scale = _coded(v, kind)
        pool["v"][at, :, slot], pool["v_scale"][at, :, slot] = codes, scale
    lo, hi = pool["bounds"].float().unbind(2)
    begun = at[slot == 0]  # blocks that begin in this call have no bounds from before
    lo, hi = lo.index_fill(0, begun, torch.inf), hi.index_fill(0, begun, -torch.inf)
    x = torch.where(torch.isfinite(k), k, 0).float()
    both = torch.stack((lo.index_reduce_(0, at, x, "amin"), hi.index_reduce_(0, at, x, "amax")), 2)
    pool["bounds"][at] = both[at].to(k.dtype)
    codes, scale = _coded(both[at].flatten(2), "int8")
    pool["bound_codes"][at], pool["bound_scale"][at] = codes.view(both[at].shape), scale


def _vectors(s, T):
    pool, page, dtype = s["pool"], s["case"]["page"], DTYPES[s["case"]["dtype"]]
    seq, pos = _places(s, T)
    at, slot = s["table"][seq, pos // page].long(), pos % page
    k, v = pool["k"][at, :, slot], pool["v"][at, :, slot]
    if pool["k_scale"] is not None:
        k, v = k.float() * pool["k_scale"][at, :, slot][..., None], v.float() * pool["v_scale"][at, :, slot][..., None]
    return k.to(dtype), v.to(dtype)


def _query_codes(q, H):
    """The queries of a key head's group as whole numbers from -127 to 127: (T, H, 2 D), for the lower bounds and the upper.
    A sum over the group of max(q lo, q hi) is the product of the bounds with the sums of the negative and the positive parts."""
    T, HG, D = q.shape
    x = torch.where(torch.isfinite(q), q, 0).view(T, H, HG // H * D)
    whole = _coded(x, "int8")[0].view(T, H, HG // H, D).long()
    parts = torch.cat((whole.clamp(max=0).sum(2), whole.clamp(min=0).sum(2)), -1)
    most = parts.abs().amax(-1, keepdim=True)
    return torch.where(most > 0, parts.double() * 127.0 / most.clamp(min=1).double(), 0.0).round()


def _search(s, k):
    """(T, heads, k) blocks for every query, ascending, -1 behind the last.  The first block and the two at the query's
    own position are always among them, the others by score: a product of whole numbers times the block's scale."""
    case, pool = s["case"], s["pool"]
    H, page, T = case["heads"], case["page"], s["q"].shape[0]
    seq, pos = _places(s, T)
    table = s["table"].long()
    B, W = table.shape
    row = torch.arange(T, device="cuda") - (torch.arange(T, device="cuda") if s["cu"] is None else s["cu"].long()[seq])
    padded = torch.zeros((B, max(_lengths(case)[0]), H, 2 * case["dim"]), dtype=torch.float64, device="cuda")
    padded[seq, row] = _query_codes(s["q"], H)
    bounds = pool["bound_codes"][table.clamp(min=0)].flatten(3).double()  # (B, W, H, 2 D)
    whole = torch.matmul(padded.transpose(1, 2), bounds.permute(0, 2, 3, 1)).transpose(1, 2)[seq, row]  # (T, H, W), exact
    score = whole.float() * pool["bound_scale"][table.clamp(min=0)].transpose(1, 2)[seq]
    block, last = torch.arange(W, device="cuda")[None, None], (pos // page)[:, None, None]
    score = torch.where((block < 1) | (block > last - 2), torch.inf, score)
    score = torch.where((block <= last) & (table[seq] >= 0)[:, None], score, -torch.inf)
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)
    best, at = best[..., :k], at[..., :k]
    at = torch.where(best > -torch.inf, at, W).sort(-1).values
    at = torch.nn.functional.pad(at, (0, k - at.shape[-1]), value=W)
    return torch.where(at < W, at, -1).to(torch.int32)


def _softmaxed(score, v):
    """Softmax over the last axis times v, and the logarithm of the sum; a row of nothing but -inf gives zeros and -inf."""
    most = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(most == -torch.inf, 0.0, most))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(p, v) / total, 0.0), (most + torch.log(total)).squeeze(-1)


def _attend(s):
    case, pool = s["case"], s["pool"]
    H, G, D, page, T, q = case["heads"], case["group"], case["dim"], case["page"], s["q"].shape[0], s["q"].float()
    seq, pos = _places(s, T)
    table, head = s["table"].long(), torch.arange(H, device="cuda")[None, :, None]
    if s["blocks"] is not None:  # every query and key head has blocks of its own
        blocks = s["blocks"].long()
        own_pages = table[seq[:, None, None], blocks.clamp(min=0)]  # (T, H, K)
        there = (blocks >= 0) & (own_pages >= 0)
        q, limit = q.view(T, H, G, D), pos[:, None, None, None]
    else:  # those of a sequence share them
        row = torch.arange(T, device="cuda") - (torch.arange(T, device="cuda") if s["cu"] is None else s["cu"].long()[seq])
        B, W = table.shape
        n = max(_lengths(case)[0])
        blocks = torch.arange(W, device="cuda").expand(B, H, W)
        own_pages = table[:, None].expand(B, H, W)
        there = own_pages >= 0
        padded, limit = q.new_zeros((B, n, H, G, D)), pos.new_full((B, n), -1)
        padded[seq, row], limit[seq, row] = q.view(T, H, G, D), pos
        q, limit = padded.permute(0, 2, 1, 3, 4).reshape(B, H, n * G, D), limit.repeat_interleave(G, 1)[:, None, :, None]
    at = own_pages.clamp(min=0)
    k, v = pool["k"][at, head].float(), pool["v"][at, head].float()  # (., H, K, page, D)
    if pool["k_scale"] is not None:
        k, v = k.mul_(pool["k_scale"][at, head][..., None]), v.mul_(pool["v_scale"][at, head][..., None])
    where = (blocks[..., None] * page + torch.arange(page, device="cuda")).flatten(2)[:, :, None]  # positions
    score = torch.matmul(q, k.flatten(2, 3).transpose(2, 3)) * D**-0.5
    score = torch.where((where <= limit) & there[..., None].expand(*there.shape, page).flatten(2)[:, :, None], score, -torch.inf)
    out, lse = _softmaxed(score, v.flatten(2, 3))
    if s["blocks"] is None:
        out, lse = out.view(B, H, n, G, D).transpose(1, 2)[seq, row], lse.view(B, H, n, G).transpose(1, 2)[seq, row]
    return out.reshape(T, H * G, D).to(DTYPES[case["dtype"]]), lse.reshape(T, H * G)


# ------------------------------------------------------------------------------------------------------- the call
def run(s):
    case, pool, cache = s["case"], s["pool"], s.get("cache")
    path, T = case["path"], s["q"].shape[0]
    if path == "add":  # and what it wrote read back, as the values that the codes stand for
        if own:
            cache.add(s["new_k"], s["new_v"], s["table"], s["lens"], cu=s["cu"])
            k, v = cache.vectors(s["table"], s["lens"], cu=s["cu"], rows=T)
        else:
            _add(s)
            k, v = _vectors(s, T)
        # the codes of the bounds are the whole numbers that a search multiplies
        return dict(k=k, v=v, **{name: pool[name] for name in ("k_scale", "v_scale", "bounds", "bound_codes", "bound_scale")})
    if path == "vectors":
        k, v = cache.vectors(s["table"], s["lens"], cu=s["cu"], rows=T) if own else _vectors(s, T)
        return dict(k=k, v=v)
    if path == "search":
        if own:
            return cache.search_blocks(s["q"], s["table"], s["lens"], case["k"], cu=s["cu"], first=1, recent=2)
        return _search(s, case["k"])
    if own:
        out, lse = cache.attend(s["q"], s["table"], s["lens"], cu=s["cu"], blocks=s["blocks"], return_lse=True)
    else:
        out, lse = _attend(s)
    return dict(out=out, lse=lse)


# ----------------------------------------------------------------------------------------------- what is expected
def work(case):
    new, lens = _lengths(case)
    H, G, D, page, T, B = case["heads"], case["group"], case["dim"], case["page"], sum(new), case["B"]
    held = 2 * D if case["kind"] == "same" else D + 4  # bytes of a row in the cache
    tables = 4 * sum(-(-n // page) for n in lens) + 8 * B
    touched = sum((n - 1) // page - (n - m) // page + 1 for n, m in zip(lens, new))
    bound_bytes = H * (2 * D + 4)
    if case["path"] == "add":  # rows in, rows of the cache out, the same rows read back; bounds are read, written and coded
        return dict(bytes=2 * T * H * (2 * D + held + 2 * D) + touched * (bound_bytes + 8 * H * D) + tables, flops=T * H * D * 8)
    if case["path"] == "vectors":
        return dict(bytes=2 * T * H * (held + 2 * D) + tables, flops=0 if case["kind"] == "same" else 2 * T * H * D)
    pairs = sum(m * ((n - m) // page + 1) + sum(range(0, m, page)) for n, m in zip(lens, new))  # (query, block) pairs, nearly
    if case["path"] == "search":
        return dict(bytes=2 * T * H * G * D + sum(-(-n // page) for n in lens) * bound_bytes + tables + 4 * T * H * case["k"],
                    flops=H * (4 * D * pairs + 4 * T * G * D))
    seen = [[min(n - m + i + 1, case["k"] * page if case["k"] else n) for i in range(m)] for n, m in zip(lens, new)]
    rows = sum(min(n, sum(x)) for n, x in zip(lens, seen))  # each row that is attended to once, at most
    if case["k"] and max(new) > 1:  # the fewest that could have been selected: the queries' blocks the same
        rows = sum(min(n, case["k"] * page + m) for n, m in zip(lens, new))
    return dict(bytes=2 * rows * H * held + 4 * T * H * G * D + 4 * T * H * G + tables + 4 * T * H * case["k"],
                flops=4 * H * G * D * sum(map(sum, seen)))


def exact(case, seed):
    """From the definitions, one sequence after the other, in 64 bits."""
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    new, lens = _lengths(case)
    cu, page, H, G, D, kind = _first(new), case["page"], case["heads"], case["group"], case["dim"], case["kind"]
    pool, table = s["pool"], s["table"].long()

    def rows_of(b, name, begin, end):  # (rows, H, D) of sequence b as they are held
        at = table[b, : -(-end // page)]
        x = pool[name][at].double()
        if kind != "same":
            x = x * pool[name + "_scale"][at].double()[..., None]
        return x.transpose(1, 2).reshape(-1, H, D)[begin:end]

    if case["path"] == "vectors":
        return {name: torch.cat([rows_of(b, name, n - m, n) for b, (n, m) in enumerate(zip(lens, new))]) for name in ("k", "v")}
    if case["path"] == "search":
        return None  # whole numbers
    if case["path"] == "add":
        got = dict(k_scale=pool["k_scale"], v_scale=pool["v_scale"])
        got = {n: None if x is None else x.double() for n, x in got.items()}
        bounds, bound_scale = pool["bounds"].double(), pool["bound_scale"].double()
        for name in ("k", "v"):
            x = s["new_" + name].double()
            if kind != "same":
                most = x.abs().amax(-1, keepdim=True)
                y = x * TOP[kind] / most.clamp(min=1e-300)
                if kind == "int8":
                    y = torch.round(y)  # halves to the even number
                else:
                    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)  # the step of e4m3 at y
                    y = torch.round(y / unit) * unit
                got[name] = y * (most / TOP[kind])
            else:
                got[name] = x
        for b, (n, m) in enumerate(zip(lens, new)):
            for i in range((n - m) // page, (n - 1) // page + 1):
                lo, hi = max(n - m, i * page), min(n, (i + 1) * page)
                x, at = s["new_k"][cu[b] + lo - (n - m) : cu[b] + hi - (n - m)].double(), table[b, i]
                least, most = x.amin(0), x.amax(0)
                if lo > i * page:  # the block had rows before
                    least, most = torch.minimum(least, bounds[at, :, 0]), torch.maximum(most, bounds[at, :, 1])
                bounds[at, :, 0], bounds[at, :, 1] = least, most
                bound_scale[at] = torch.maximum(least.abs(), most.abs()).amax(-1) / 127.0
            if kind != "same":
                pos = torch.arange(n - m, n, device="cuda")
                for name in ("k", "v"):
                    step = s["new_" + name][cu[b] : cu[b + 1]].double().abs().amax(-1) / TOP[kind]
                    got[name + "_scale"][table[b, pos // page], :, pos % page] = step
        return dict(got, bounds=bounds, bound_codes=None, bound_scale=bound_scale)
    if sum(m * n for m, n in zip(new, lens)) * H * G > 2_000_000_000:
        return None
    outs, lses = [], []
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = rows_of(b, "k", 0, n), rows_of(b, "v", 0, n)
        q = s["q"][cu[b] : cu[b + 1]].double().view(m, H, G, D)
        score = torch.einsum("mhgd,nhd->mhgn", q, k) / D**0.5
        seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - m, n, device="cuda")[:, None]
        seen = seen[:, None].expand(m, H, n)
        if s["blocks"] is not None:
            listed_blocks = torch.zeros((m, H, table.shape[1] + 1), dtype=torch.bool, device="cuda")
            listed_blocks.scatter_(2, s["blocks"][cu[b] : cu[b + 1]].long() % (table.shape[1] + 1), True)
            seen = seen & listed_blocks[..., torch.arange(n, device="cuda") // page]
        score = score.masked_fill(~seen[:, :, None], -torch.inf)
        lses.append(torch.logsumexp(score, -1).reshape(m, H * G))
        outs.append(torch.einsum("mhgn,nhd->mhgd", torch.softmax(score, -1), v).reshape(m, H * G, D))
    return dict(out=torch.cat(outs), lse=torch.cat(lses))
