"""What a server does around the key/value cache: what is measured, and its plain forms.

`rotate` turns queries and keys by their positions before they are added and attended to; `add` writes rows to a cache that
holds them in 4 bits (kind "int4x32") and reads them back; `attend` is attention over such a cache, for single rows and for
prompts, over listed blocks or all; `branch` is a step of sequences that share pages: each goes on from one of the last step's
(fork), the last step's are given back (free) and the new ones get room for their next rows, with a page of their own where they
share one (extend); `compact` moves the pages in use to the front of the memory.

A batch is `KvCache`'s: `table[b, i]` is the page of block i of sequence b, `lens[b]` its rows, and a call is about its last ones.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUP4 = 32  # components that share a scale
LARGEST = 9216.0  # scale: 7 times it is in fp16's range


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of a server with 24 requests, halves of the whole head turned
        dict(name="rotate_tokens", path="rotate", dtype="bf16", B=24, new=1, ctx=4000, heads=8, group=4, dim=128, part=128, layout="half", factor=1.0, original=0),
        # prompts far beyond the context that a model was trained on, neighbours turned in half of the head
        dict(name="rotate_prompts", path="rotate", dtype="fp16", B=6, new=2900, ctx=130000, heads=8, group=4, dim=128, part=64, layout="pairs", factor=16.0, original=8192),
        # one decoding step's rows into the cache
        dict(name="add_tokens", path="add", dtype="bf16", B=24, new=1, ctx=4000, page=64, heads=8, group=4, dim=128),
        # the prompts of six requests, of different lengths, at once
        dict(name="add_prompts", path="add", dtype="bf16", B=6, new=2900, ctx=2900, page=64, heads=8, group=4, dim=128),
        # a decoding step of one request over the blocks that were found for it
        dict(name="attend_one", path="attend", dtype="bf16", B=1, new=1, ctx=50000, page=64, heads=8, group=4, dim=128, k=32),
        # a full batch's decoding step over listed blocks
        dict(name="attend_batch", path="attend", dtype="bf16", B=64, new=1, ctx=20000, page=64, heads=8, group=8, dim=128, k=40),
        # a decoding step over whole sequences, heads of 96, smaller pages
        dict(name="attend_all", path="attend", dtype="fp16", B=12, new=1, ctx=30000, page=32, heads=8, group=5, dim=96, k=0),
        # a piece of two prompts over everything before it
        dict(name="attend_prompt", path="attend", dtype="bf16", B=2, new=1500, ctx=6000, page=64, heads=8, group=4, dim=128, k=0),
        # beams of two requests: four sequences each, of which the best go on
        dict(name="branch_beams", path="branch", dtype="bf16", B=8, share=4, ctx=900, more=1, page=16, heads=4, dim=128, layers=2, pages=2000),
        # samples of 32 requests, eight of each, every one with drafted rows of its own
        dict(name="branch_samples", path="branch", dtype="fp16", B=256, share=8, ctx=4010, more=7, page=32, heads=2, dim=64, layers=2, pages=30000),
        # a small cache after requests of different lengths have ended
        dict(name="compact_small", path="compact", dtype="bf16", B=12, ctx=1500, live=0.6, page=16, heads=4, dim=64, layers=1, pages=1500),
        # a large one
        dict(name="compact_large", path="compact", dtype="bf16", B=100, ctx=8000, live=0.5, page=64, heads=4, dim=128, layers=1, pages=20000),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    path = rng.choice(["rotate", "add", "attend", "attend", "attend", "branch", "compact"])
    case = dict(path=path, dtype=rng.choice(["bf16", "fp16"]), dim=rng.choice([64, 96, 128, 128]))
    if path in ("branch", "compact"):
        case |= dict(page=rng.choice([16, 32, 64, 128]), heads=rng.choice([1, 2, 3, 4]), layers=rng.choice([1, 1, 2, 3]), B=_log(rng, 1, 256))
        page_bytes = 4 * case["heads"] * case["page"] * case["dim"] * case["layers"]
        case["ctx"] = _log(rng, 1, 8000)
        if path == "branch":
            case |= dict(share=rng.choice([1, 2, 4, 7, 8]), more=rng.choice([0, 1, 1, rng.randint(2, 40), 700]))
            case["ctx"] = max(1, min(case["ctx"], 400_000_000 // page_bytes * case["page"] // case["B"]))
            case["pages"] = case["B"] * ((case["ctx"] + 2 * case["more"]) // case["page"] + 3) + rng.randint(0, 500)
        else:
            case["live"] = rng.choice([0.05, 0.3, 0.5, 0.8, 1.0])
            case["ctx"] = max(1, min(case["ctx"], 1_200_000_000 // page_bytes * case["page"] // case["B"]))
            case["pages"] = int(case["B"] * -(-case["ctx"] // case["page"]) / case["live"]) + rng.randint(0, 50)
            case["pages"] = max(case["B"] * -(-case["ctx"] // case["page"]), min(case["pages"], 2_600_000_000 // page_bytes))
        return case
    case |= dict(heads=rng.choice([1, 2, 4, 8, 8]), group=rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]))
    row = case["heads"] * case["dim"]
    if path == "rotate":
        case["new"] = rng.choice([1, _log(rng, 1, 20_000)])
        case["B"] = _log(rng, 1, max(1, min(256, 80_000_000 // (row * (case["group"] + 1) * case["new"]))))
        case |= dict(ctx=case["new"] + _log(rng, 1, 1_000_000), part=rng.choice([16, 32, 64, case["dim"], case["dim"]]), layout=rng.choice(["half", "pairs"]))
        case |= rng.choice([dict(factor=1.0, original=0), dict(factor=4.0, original=0), dict(factor=8.0, original=4096)])
        return case
    case["page"] = rng.choice([16, 32, 64, 64, 128])
    if path == "add":
        case["new"] = rng.choice([1, _log(rng, 1, 20_000)])
        case["B"] = _log(rng, 1, max(1, min(256, 16_000_000 // (row * case["new"]))))
        case["ctx"] = case["new"] + rng.choice([0, _log(rng, 1, 2000)])
        case["B"] = max(1, min(case["B"], 60_000_000 // (row * case["ctx"])))
        return case
    case["new"] = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 1000)])
    case["ctx"] = case["new"] + _log(rng, 1, 60_000)
    dense = rng.random() < 0.4
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
    return new, [n + (case["ctx"] - case["new"]) * (16 - (b * 37) % 11) // 16 for b, n in enumerate(new)]


def _first(x):
    """Where each of the numbers x begins when they stand one behind the other."""
    at = [0]
    for n in x:
        at.append(at[-1] + n)
    return at


def _frequencies(case):
    """Radians a position for each pair, and what the turned components are multiplied by."""
    w = [10000.0 ** (-2 * i / case["part"]) for i in range(case["part"] // 2)]
    f, original = case["factor"], case["original"]
    if not original:
        return [x / f for x in w], 1.0
    keep = [min(max((original * x / (2 * math.pi) - 1.0) / 31.0, 0.0), 1.0) for x in w]  # below one turn in `original` positions: interpolated; above 32: not
    return [x * (g + (1 - g) / f) for x, g in zip(w, keep)], 0.1 * math.log(f) + 1.0


# --------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(int(seed))
    randn = lambda *n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    dtype, D = DTYPES[case["dtype"]], case["dim"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    s = dict(case=case)
    if case["path"] in ("branch", "compact"):
        return _prepare_pages(s, g, randn, dtype)
    H, G, B = case["heads"], case["group"], case["B"]
    new, lens = _lengths(case)
    s |= dict(lens=i32(lens), cu=i32(_first(new)) if case["new"] > 1 else None)
    T = sum(new)
    channel = 2.0 * randn(H, D) * (torch.rand((H, D), generator=g, device="cuda") < 0.1)  # some channels of keys are far from zero
    rows = randn(T, H * (G + 2), D)  # queries, and new keys and values, are parts of one projection's rows
    rows[:, H * G : H * (G + 1)] += channel
    s["rows"] = rows.to(dtype)
    s["q"], s["k"], s["v"] = s["rows"].split([H * G, H, H], 1)
    if case["path"] == "rotate":
        w, s["amplitude"] = _frequencies(case)
        s["w"] = torch.tensor(w, dtype=torch.float64, device="cuda")
        if own:  # the handle that a program keeps
            import ferrolm_b200 as fv

            s["rotary"] = fv.Rotary(D, part=case["part"], layout=case["layout"], factor=case["factor"], original=case["original"] or None)
        return s
    page = case["page"]
    blocks = [-(-n // page) for n in lens]
    W, P = max(blocks), sum(blocks) + 3
    at, of = _first(blocks), torch.randperm(P, generator=g, device="cuda").to(torch.int32)  # pages are handed out in no order
    table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(blocks):
        table[b, :n] = of[at[b] : at[b] + n]
    s["table"] = table
    k = randn(P, H, page, D) + channel[:, None]
    bounds = torch.stack((k.amin(2), k.amax(2)), 2).to(dtype)
    codes, scale = _coded8(bounds.flatten(2))
    pool = dict(bounds=bounds, bound_codes=codes.view(bounds.shape), bound_scale=scale)
    pool["k"], pool["k_scale"] = _coded4(k.to(dtype))
    pool["v"], pool["v_scale"] = _coded4(randn(P, H, page, D).to(dtype))
    s["pool"] = pool
    if case["path"] == "attend":
        s["blocks"] = _some_blocks(s, g, T) if case["k"] else None
    if own:
        import ferrolm_b200 as fv

        s["cache"] = fv.KvCache(P, H, D, page_size=page, dtype=dtype, kind="int4x32", buffers=pool)
    return s


def _some_blocks(s, g, T):
    """Ascending blocks for every row and key head, the first and the last two among them; the rows of 32 positions look alike."""
    case, (seq, pos) = s["case"], _places(s, T)
    W = s["table"].shape[1]
    like = torch.rand((case["B"], int(max(_lengths(case)[0])) // 32 + 2, case["heads"], W), generator=g, device="cuda")
    row = torch.arange(T, device="cuda") - (torch.arange(T, device="cuda") if s["cu"] is None else s["cu"].long()[seq])
    score = like[seq, row // 32] + 0.1 * torch.rand((T, case["heads"], W), generator=g, device="cuda")
    block, last = torch.arange(W, device="cuda")[None, None], (pos // case["page"])[:, None, None]
    score = torch.where((block < 1) | (block > last - 2), torch.inf, score)
    best, at = torch.sort(torch.where(block <= last, score, -torch.inf), dim=-1, descending=True, stable=True)
    best, at = best[..., : case["k"]], at[..., : case["k"]]
    at = torch.where(best > -torch.inf, at, W).sort(-1).values
    at = torch.nn.functional.pad(at, (0, case["k"] - at.shape[-1]), value=W)
    return torch.where(at < W, at, -1).to(torch.int32)


def _prepare_pages(s, g, randn, dtype):
    case = s["case"]
    B, page, P, H, D = case["B"], case["page"], case["pages"], case["heads"], case["dim"]
    if case["path"] == "branch":  # sequences of one request share all but the last quarter of their blocks
        share = case["share"]
        lens = [max(1, case["ctx"] * (16 - (b // share * 37) % 11) // 16 - (b % share) % 3) for b in range(B)]
    else:
        share = 1
        lens = [max(1, case["ctx"] * (16 - (b * 37) % 11) // 16) for b in range(B)]
    blocks = [-(-n // page) for n in lens]
    W = max(blocks) + (-(-case.get("more", 0) // page) + 1 if case["path"] == "branch" else 0)
    number = [[-1] * W for _ in range(B)]
    used = 0
    for b, n in enumerate(blocks):
        common = 0 if b % share == 0 else 3 * min(n, blocks[b - 1]) // 4
        number[b][:n] = number[b - 1][:common] + list(range(used, used + n - common))
        used += n - common
    of = torch.cat((torch.randperm(P, generator=g, device="cuda"), torch.tensor([-1], device="cuda")))  # pages in use are anywhere
    s["table"] = of[torch.tensor(number, device="cuda")].to(torch.int32)
    s["refs"] = torch.zeros(P + 1, dtype=torch.int32, device="cuda").index_add_(0, (s["table"].long() % (P + 1)).flatten(), torch.ones(B * W, dtype=torch.int32, device="cuda"))[:P].clone()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["more"] = torch.full((B,), case.get("more", 0), dtype=torch.int32, device="cuda")
    s["parents"] = torch.randint(0, max(1, share), (B,), generator=g, device="cuda").to(torch.int32) + torch.arange(B, dtype=torch.int32, device="cuda") // share * share
    s["parents"].clamp_(max=B - 1)
    s["pools"] = []
    for _ in range(case["layers"]):
        k, v = (torch.empty((P, H, page, D), dtype=dtype, device="cuda").normal_(generator=g) for _ in range(2))
        bounds = torch.stack((k.amin(2), k.amax(2)), 2)
        codes, scale = _coded8(bounds.flatten(2))
        s["pools"].append(dict(k=k, v=v, bounds=bounds, bound_codes=codes.view(bounds.shape), bound_scale=scale))
    if own:
        import ferrolm_b200 as fv

        caches = [fv.KvCache(P, H, D, page_size=page, dtype=dtype, buffers=pool) for pool in s["pools"]]
        s["pages"] = fv.KvPages(caches)
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


def _rotate(s, x):
    """Angles of far positions need 64 bits."""
    part, half = s["case"]["part"], s["case"]["part"] // 2
    angle = _places(s, x.shape[0])[1].double()[:, None, None] * s["w"]
    c, d = (angle.cos() * s["amplitude"]).float(), (angle.sin() * s["amplitude"]).float()
    y = x.float()
    if s["case"]["layout"] == "half":
        a, b = y[..., :half], y[..., half:part]
        turned = torch.cat((a * c - b * d, b * c + a * d), -1)
    else:
        a, b = y[..., 0:part:2], y[..., 1:part:2]
        turned = torch.stack((a * c - b * d, b * c + a * d), -1).flatten(2)
    return torch.cat((turned, y[..., part:]), -1).to(x.dtype)


def _coded8(x):
    """Rows as whole numbers to 127, and their scales.  The quotient lies next to the border of two codes too often for 32 bits."""
    most = x.float().abs().amax(-1, keepdim=True)
    y = torch.where(most > 0, x.double() * 127.0 / most.double(), 0.0)
    return y.round().to(torch.int8), (most / torch.full_like(most, 127.0)).squeeze(-1)


def _coded4(x):
    """Rows in 4 bits: for 32 components the smallest scale of 4 significant bits that 7 times is not below any of them, and whole
    numbers to 7, 8 added.  16 bits of a row hold four neighbouring components; the groups' first four stand before their second four."""
    y = x.double().unflatten(-1, (-1, GROUP4))
    t = y.abs().amax(-1, keepdim=True) / 7.0
    unit = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0**-14))).clamp(min=-14.0) - 3.0)  # the step of scales at t
    scale = ((t / unit).ceil() * unit).clamp(max=LARGEST)
    code = torch.where(scale > 0, (y / torch.where(scale > 0, scale, 1.0)).round().clamp(-7, 7), 0.0) + 8.0
    byte = (scale.squeeze(-1).half().view(torch.int16) >> 7).to(torch.uint8)
    code = code.to(torch.uint8).unflatten(-1, (8, 4)).transpose(-3, -2).flatten(-3)
    return code[..., 0::2] | code[..., 1::2] << 4, byte


def _values4(packed, byte):
    scale = (byte.to(torch.int16) << 7).view(torch.float16).float()
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).unflatten(-1, (8, -1, 4)).transpose(-3, -2).flatten(-2)
    return ((code.float() - 8.0) * scale[..., None]).flatten(-2)


def _add(s):
    pool, page = s["pool"], s["case"]["page"]
    k, v = s["k"], s["v"]
    seq, pos = _places(s, k.shape[0])
    at, slot = s["table"][seq, pos // page].long(), pos % page
    for name, x in (("k", k), ("v", v)):
        pool[name][at, :, slot], pool[name + "_scale"][at, :, slot] = _coded4(x)
    lo, hi = pool["bounds"].float().unbind(2)
    begun = at[slot == 0]  # blocks that begin in this call have no bounds from before
    lo, hi = lo.index_fill(0, begun, torch.inf), hi.index_fill(0, begun, -torch.inf)
    x = torch.where(torch.isfinite(k), k, 0).float()
    both = torch.stack((lo.index_reduce_(0, at, x, "amin"), hi.index_reduce_(0, at, x, "amax")), 2)
    pool["bounds"][at] = both[at].to(k.dtype)
    codes, scale = _coded8(both[at].flatten(2))
    pool["bound_codes"][at], pool["bound_scale"][at] = codes.view(both[at].shape), scale
    dtype = DTYPES[s["case"]["dtype"]]
    return tuple(_values4(pool[n][at, :, slot], pool[n + "_scale"][at, :, slot]).to(dtype) for n in ("k", "v"))


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
        pages = table[seq[:, None, None], blocks.clamp(min=0)]  # (T, H, K)
        there = (blocks >= 0) & (pages >= 0)
        q, limit = q.view(T, H, G, D), pos[:, None, None, None]
    else:  # those of a sequence share them
        row = torch.arange(T, device="cuda") - (torch.arange(T, device="cuda") if s["cu"] is None else s["cu"].long()[seq])
        B, W = table.shape
        n = max(_lengths(case)[0])
        blocks = torch.arange(W, device="cuda").expand(B, H, W)
        pages = table[:, None].expand(B, H, W)
        there = pages >= 0
        padded, limit = q.new_zeros((B, n, H, G, D)), pos.new_full((B, n), -1)
        padded[seq, row], limit[seq, row] = q.view(T, H, G, D), pos
        q, limit = padded.permute(0, 2, 1, 3, 4).reshape(B, H, n * G, D), limit.repeat_interleave(G, 1)[:, None, :, None]
    at = pages.clamp(min=0)
    k, v = (_values4(pool[n][at, head], pool[n + "_scale"][at, head]) for n in ("k", "v"))  # (., H, K, page, D)
    where = (blocks[..., None] * page + torch.arange(page, device="cuda")).flatten(2)[:, :, None]  # positions
    score = torch.matmul(q, k.flatten(2, 3).transpose(2, 3)) * D**-0.5
    score = torch.where((where <= limit) & there[..., None].expand(*there.shape, page).flatten(2)[:, :, None], score, -torch.inf)
    out, lse = _softmaxed(score, v.flatten(2, 3))
    if s["blocks"] is None:
        out, lse = out.view(B, H, n, G, D).transpose(1, 2)[seq, row], lse.view(B, H, n, G).transpose(1, 2)[seq, row]
    return out.reshape(T, H * G, D).to(DTYPES[case["dtype"]]), lse.reshape(T, H * G)


def _copied(s, src, dst):
    for pool in s["pools"]:
        for x in pool.values():
            x[dst] = x[src]


def _counted(refs, pages, by):
    """`by` added to the count of every page in `pages` (-1: none)."""
    P = refs.shape[0]
    return torch.cat((refs, refs.new_zeros(1))).index_add(0, torch.where(pages >= 0, pages, P).flatten(), torch.full((pages.numel(),), by, dtype=refs.dtype, device="cuda"))[:P]


def _branch(s):
    case, P, page = s["case"], s["refs"].shape[0], s["case"]["page"]
    W, refs = s["table"].shape[1], s["refs"]
    block = torch.arange(W, device="cuda")[None]
    # fork: the parents' blocks, up to their rows
    lens = s["lens"][s["parents"].long()].long()
    table = torch.where(block * page < lens[:, None], s["table"][s["parents"].long()], -1).long()
    refs = _counted(_counted(refs, table, 1), s["table"].long(), -1)  # and the last step's are given back
    # extend: blocks that rows come to.  One that others have too becomes a page of its own, but for its first holder where nobody else is left.
    to = (block >= (lens // page)[:, None]) & (block * page < (lens + s["more"])[:, None])
    shared = to & (table >= 0) & (refs[table.clamp(min=0)] > 1)
    here = torch.where(shared, table, P).flatten()
    left = torch.cat((refs, refs.new_ones(1))).long()
    left = left - torch.bincount(here, minlength=P + 1)
    order = torch.arange(here.numel(), device="cuda")
    first = torch.full((P + 1,), here.numel(), device="cuda").scatter_reduce(0, here, order, "amin")
    stays = shared & ((left[here] == 0) & (first[here] == order)).view(shared.shape)
    take = to & ((table < 0) | shared) & ~stays
    free = torch.sort(refs > 0, stable=True).indices  # the free pages first, the lowest before the others
    rank = (take.flatten().cumsum(0) - 1).view(take.shape)
    enough = (refs == 0).sum() >= take.sum()
    missing = torch.where(enough, 0, take.sum() - (refs == 0).sum()).to(torch.int32)
    take = take & enough
    got = free[rank.clamp(0, P - 1)]
    moved = take & shared
    refs = _counted(_counted(refs, torch.where(moved, table, -1), -1), torch.where(take, got, -1), 1)
    _copied(s, table[moved], got[moved])
    return dict(table=torch.where(take, got, table).to(torch.int32), refs=refs, missing=missing)


def _compact(s):
    refs, table, P = s["refs"], s["table"].long(), s["refs"].shape[0]
    live = refs > 0
    n, page = live.sum(), torch.arange(P, device="cuda")
    src, dst = page[live & (page >= n)], page[~live & (page < n)]  # as many of the one as of the other
    to = torch.where(live, page, -1)
    to[src] = dst
    _copied(s, src, dst)
    refs = refs.clone()
    refs[dst] = refs[src]
    refs[src] = 0
    return dict(table=torch.where(table >= 0, to[table.clamp(min=0)], -1).to(torch.int32), refs=refs, used=n.to(torch.int32))


# ------------------------------------------------------------------------------------------------------- the call
def run(s):
    case, path = s["case"], s["case"]["path"]
    if path == "rotate":
        q, k = s["rotary"].rotate(s["q"], s["k"], lens=s["lens"], cu=s["cu"]) if own else (_rotate(s, s["q"]), _rotate(s, s["k"]))
        return dict(q=q, k=k)
    if path == "add":  # and what it wrote read back, as the values that the codes stand for
        pool = s["pool"]
        if own:
            s["cache"].add(s["k"], s["v"], s["table"], s["lens"], cu=s["cu"])
            k, v = s["cache"].vectors(s["table"], s["lens"], cu=s["cu"], rows=s["k"].shape[0])
        else:
            k, v = _add(s)
        # the codes of the bounds are the whole numbers that a search multiplies
        return dict(k=k, v=v, **{name: pool[name] for name in ("bounds", "bound_codes", "bound_scale")})
    if path == "attend":
        if own:
            out, lse = s["cache"].attend(s["q"], s["table"], s["lens"], cu=s["cu"], blocks=s["blocks"], return_lse=True)
        else:
            out, lse = _attend(s)
        return dict(out=out, lse=lse)
    # a step begins from the counts and the table that the program has
    if not own:
        got = _branch(s) if path == "branch" else _compact(s)
    else:
        pages, table = s["pages"], s["table"].clone()
        pages.refs.copy_(s["refs"])
        if path == "branch":
            last, table = table, pages.fork(table, s["lens"], s["parents"])
            pages.free(last)
            pages.extend(table, s["lens"][s["parents"]], s["more"])
            got = dict(table=table, refs=pages.refs, missing=pages.missing)
        else:
            pages.compact(table)
            got = dict(table=table, refs=pages.refs, used=pages.used)
    return dict(got, layers=[{n: pool[n] for n in ("k", "v", "bounds", "bound_codes", "bound_scale")} for pool in s["pools"]])


# ----------------------------------------------------------------------------------------------- what is expected
def work(case):
    D, B = case["dim"], case["B"]
    if case["path"] in ("branch", "compact"):
        page_bytes = case["layers"] * case["heads"] * (4 * case["page"] * D + 4 * D + 2 * D + 4)
        if case["path"] == "branch":
            n = min(case["share"], B)
            alone = (1 - (1 - 1 / n) ** n) * n  # parents that somebody goes on from; the others' pages are copied
            partial = case["ctx"] % case["page"] != 0 and case["more"] > 0
            W = -(-case["ctx"] // case["page"])
            return dict(bytes=2 * page_bytes * (B / n * (n - alone) if partial else 0) + 3 * 4 * B * W + 12 * B + 4 * case["pages"], flops=0)
        blocks = sum(-(-max(1, case["ctx"] * (16 - (b * 37) % 11) // 16) // case["page"]) for b in range(B))
        return dict(bytes=2 * page_bytes * blocks * (1 - min(1.0, blocks / case["pages"])) + 8 * case["pages"] + 8 * blocks, flops=0)
    H, G = case["heads"], case["group"]
    new, lens = _lengths(case)
    T = sum(new)
    if case["path"] == "rotate":
        return dict(bytes=4 * T * H * (G + 1) * D + 8 * B, flops=3 * T * H * (G + 1) * case["part"])
    page, held = case["page"], D // 2 + D // 32  # bytes of a row in the cache
    tables = 4 * sum(-(-n // page) for n in lens) + 8 * B
    if case["path"] == "add":  # rows in, rows of the cache out, the same rows read back; bounds are read, written and coded
        touched = sum((n - 1) // page - (n - m) // page + 1 for n, m in zip(lens, new))
        return dict(bytes=2 * T * H * (2 * D + held + 2 * D) + touched * H * (10 * D + 4) + tables, flops=T * H * D * 8)
    seen = [m * (n - m) + m * (m + 1) // 2 if not case["k"] else sum(min(n - m + i + 1, case["k"] * page) for i in range(m)) for n, m in zip(lens, new)]
    rows = sum(min(n, x) for n, x in zip(lens, seen))  # each row that is attended to once, at most
    if case["k"] and max(new) > 1:  # the fewest that could have been selected: the queries' blocks the same
        rows = sum(min(n, case["k"] * page + m) for n, m in zip(lens, new))
    return dict(bytes=2 * rows * H * held + 4 * T * H * G * D + 4 * T * H * G + tables + 4 * T * H * case["k"], flops=4 * H * G * D * sum(seen))


def exact(case, seed):
    """From the definitions, one sequence after the other, in 64 bits."""
    if case["path"] in ("branch", "compact"):
        return None  # nothing is computed: whole numbers, and pages that are moved
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    new, lens = _lengths(case)
    cu, H, G, D = _first(new), case["heads"], case["group"], case["dim"]
    if case["path"] == "rotate":  # a turn is a product of complex numbers
        w, amplitude = _frequencies(case)
        half = case["part"] // 2
        pos = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, new)]).double()
        turn = torch.polar(torch.full((len(pos), half), amplitude, dtype=torch.float64, device="cuda"), pos[:, None] * torch.tensor(w, dtype=torch.float64, device="cuda"))[:, None]
        got = {}
        for name in ("q", "k"):
            x = s[name].double()
            i = torch.arange(half, device="cuda")
            i, j = (i, i + half) if case["layout"] == "half" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., i], x[..., j]) * turn
            x[..., i], x[..., j] = z.real, z.imag
            got[name] = x
        return got
    page, pool, table = case["page"], s["pool"], s["table"].long()

    def rows_of(b, name, end):  # (rows, H, D) of sequence b as they are held, from position 0 on
        at = table[b, : -(-end // page)]
        raw, scale = pool[name][at].to(torch.int64), torch.ldexp((8 + pool[name + "_scale"][at] % 8).double(), pool[name + "_scale"][at].long() // 8 - 18)
        small = pool[name + "_scale"][at] < 8
        scale = torch.where(small, pool[name + "_scale"][at].double() * 2.0**-17, scale)
        x = torch.zeros((*raw.shape[:-1], D), dtype=torch.float64, device="cuda")
        for c in range(D):
            group, u, e = c // 32, c % 32 // 4, c % 4
            place = (u * (D // 32) + group) * 4 + e
            x[..., c] = ((raw[..., place // 2] >> 4 * (place % 2) & 15) - 8) * scale[..., group]
        return x.transpose(1, 2).reshape(-1, H, D)[:end]

    if case["path"] == "add":
        got, bounds, bound_scale = {}, pool["bounds"].double(), pool["bound_scale"].double()
        for name in ("k", "v"):
            x = s[name].double().view(-1, H, D // 32, 32)
            t = x.abs().amax(-1, keepdim=True) / 7
            grid = torch.cat((torch.arange(8, device="cuda") * 2.0**-17, (torch.arange(8, 16, device="cuda") * torch.exp2(torch.arange(-17, 14, device="cuda").double())[:, None]).flatten()))
            scale = grid[torch.searchsorted(grid, t).clamp(max=int(torch.searchsorted(grid, LARGEST)))]
            got[name] = (torch.round(x / scale.clamp(min=2.0**-17)).clamp(-7, 7) * scale).flatten(2)
        for b, (n, m) in enumerate(zip(lens, new)):
            for i in range((n - m) // page, (n - 1) // page + 1):
                lo, hi = max(n - m, i * page), min(n, (i + 1) * page)
                x, at = s["k"][cu[b] + lo - (n - m) : cu[b] + hi - (n - m)].double(), table[b, i]
                least, most = x.amin(0), x.amax(0)
                if lo > i * page:  # the block had rows before
                    least, most = torch.minimum(least, bounds[at, :, 0]), torch.maximum(most, bounds[at, :, 1])
                bounds[at, :, 0], bounds[at, :, 1] = least, most
                bound_scale[at] = torch.maximum(least.abs(), most.abs()).amax(-1) / 127.0
        return dict(got, bounds=bounds, bound_codes=None, bound_scale=bound_scale)
    if sum(m * n for m, n in zip(new, lens)) * H * G > 2_000_000_000:
        return None
    outs, lses = [], []
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = rows_of(b, "k", n), rows_of(b, "v", n)
        q = s["q"][cu[b] : cu[b + 1]].double().view(m, H, G, D)
        score = torch.einsum("mhgd,nhd->mhgn", q, k) / D**0.5
        seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - m, n, device="cuda")[:, None]
        seen = seen[:, None].expand(m, H, n)
        if s["blocks"] is not None:
            marks = torch.zeros((m, H, table.shape[1] + 1), dtype=torch.bool, device="cuda")
            marks.scatter_(2, s["blocks"][cu[b] : cu[b + 1]].long() % (table.shape[1] + 1), True)
            seen = seen & marks[..., torch.arange(n, device="cuda") // page]
        score = score.masked_fill(~seen[:, :, None], -torch.inf)
        lses.append(torch.logsumexp(score, -1).reshape(m, H * G))
        outs.append(torch.einsum("mhgn,nhd->mhgd", torch.softmax(score, -1), v).reshape(m, H * G, D))
    return dict(out=torch.cat(outs), lse=torch.cat(lses))
